// Products of two matrices on the matrix units, tile by tile:  C[m][n] = sum_k A(m, k) B(n, k),  rows of bf16 or fp32, sums in fp32.
//
// Either operand lies with its k side by side ("rows": element (i, k) at i ld + k) or its rows side by side ("columns": at k ld + i), so that the
// products of a layer's forward pass (rows, rows), of the gradient of its input (rows, columns) and of its weight (columns, columns) all
// read their operands as they lie in memory.
//
// A workgroup takes a tile of BM x BN.  128 bytes of k of both operands (64 bf16 or 32 fp32 numbers: a line of the caches) are a step; two
// steps are kept in LDS, filled by loads that write LDS directly, without registers.  A wave goes through a step in four parts and reads the
// operands of the next part while the matrix units work on one.  A step needs one barrier, before its last part: behind it the loads of
// the next step have landed for all waves, and the present step's place, which all have read, is free for the one after.
//
// Layout of a step in LDS: pieces of 16 bytes, a row of an operand that lies in rows as eight pieces, a k of one that lies in columns as
// BM / 8 (BM / 4) pieces, in either case with the piece's number changed by an exclusive or (`swizzle`) so that the sixteen lanes that
// read at one time find sixteen different places among the banks.  (The direct loads write lane after lane, so the change is made to the
// address that a lane reads from.)
//
// The 16 x 16 results are arranged so that a lane holds eight neighbouring columns of C of one row, and two fragments together are 16-byte stores
// without a turn through LDS.  B stands first in the matrix instructions, so that its index runs along a lane's four numbers.  Where B lies
// in rows, its fragment f is made of rows 32 (f / 2) + 8 (j / 4) + 4 (f % 2) + j % 4, j < 16, of a wave's part; where it lies in columns such
// fragments would be read at half the rate (pieces of 8 bytes, 16 apart), and neighbouring ones' results change places at the end instead.
//
// Bound by LDS: a step of 256 x 256 of bf16 rows keeps the matrix units busy for 2048 cycles, and its loads (16 cycles a KB) and reads (10 a KB of 16-byte
// ones, 13 of transposing ones) with them take 2950 cycles with both operands in rows, 3200 with one and 3700 with both in columns; under a long load
// by power too (clocks of 1.4 to 2.1 GHz).  8192 rows of 5632 by 2048 columns: 145 us, 1.30 PFLOP/s, and 160 us among many of them, where a large library
// product reaches 1.43.  fp32 rows are bound by the matrix units: 127 to 143 TFLOP/s where tiles fill the chip, the library's 153.
//
// Whatever lies behind a matrix (rows behind the last one, k behind the end) is read as zero: by the bounds of the buffer for whole rows,
// by an address beyond all bounds for the rest of a row.
#pragma once
#include <type_traits>

#include "pal_common.h"

namespace pal {

struct TileOperand {
  const char* p;       // element (0, 0)
  const char* p2;      // second matrix of the same shape (NULL: none): see TileArgs
  int64_t ld;          // bytes from row to row (lies in rows) or from k to k (lies in columns)
  int32_t rows;        // m or n
};

// What a forward pass keeps of the two factors g and u of a gated product, [rows][ld] each: of fp32 rows the numbers, of bf16 rows 16 bits a
// number as well, but more exactly than in bf16 (see Kept8).
struct Kept {
  void *gate, *up;           // NULL: not kept
};

// up to three products over the same k in one launch
struct TileProduct {
  TileOperand a, b;
  void* c;             // [m][n], rows ldc numbers apart
  float* part;         // [splits][m][n] where k is split (kTileGated: [splits][m][2 n], the first matrix' columns and then the second's)
  int64_t ldc;
  int32_t first;       // its first tile
  int32_t tiles_n;
};
struct TileArgs {
  TileProduct prod[3];
  int32_t n_prod;
  int32_t k;           // of one matrix; twice as much is walked where both operands have a second one (kind kTileTwice)
  int32_t tiles;       // all products'
  int32_t splits;      // of k, each of a whole number of steps
  int32_t split_steps;
  // for the feed-forward block's kinds
  Kept kept;
  void* c2;            // [m][n] beside C, rows as far apart
  int32_t act;
  int32_t used;        // columns of C from here on are padding
};

enum TileKind {
  kTilePlain = 0,
  kTileGated,   // b has two matrices, half of a tile's columns from each: C = act(A B^T) (A B2^T), both factors kept beside it if asked
  kTileGrad,    // D = A B^T is the gradient of such a C: from its kept factors the gradients of both (c, c2)
  kTileTwice,   // A B^T + A2 B2^T
};

// ---------------------------------------------------------------------------------------------------------- activations
enum { kActSilu = PAL_ACT_SILU, kActGelu = PAL_ACT_GELU, kActGeluTanh = PAL_ACT_GELU_TANH, kActRelu = PAL_ACT_RELU };

__device__ __forceinline__ float act_logistic(float x) { return fast_rcp(1.f + __expf(-x)); }
template <bool GRAD>
__device__ __forceinline__ void act_silu(float g, float& a, float& d) {
  const float f = act_logistic(g);
  a = g * f;
  if (GRAD) d = f * fmaf(g, 1.f - f, 1.f);
}
// (erfc: 1 + erf(-x) has no bits left from x = 4 on.  The fp32 training step of 1503 rows, 771 -> 2058 -> 771: 512 us with erf, 516 so.)
template <bool GRAD>
__device__ __forceinline__ void act_gelu(float g, float& a, float& d) {
  const float f = 0.5f * erfcf(g * -0.70710678118654752f);
  a = g * f;
  if (GRAD) d = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), f);
}
template <bool GRAD>
__device__ __forceinline__ void act_gelu_tanh(float g, float& a, float& d) {
  // (1 + tanh(z / 2)) / 2 is the logistic function of z
  const float g2 = g * g, f = act_logistic(1.5957691216057308f * g * fmaf(0.044715f, g2, 1.f));
  a = g * f;
  if (GRAD) {
    const float s = f * (1.f - f);
    d = s > 0.f ? fmaf(1.5957691216057308f * g * s, fmaf(0.134145f, g2, 1.f), f) : f;   // (no 0 times infinity far out)
  }
}
template <bool GRAD>
__device__ __forceinline__ void act_relu(float g, float& a, float& d) {
  a = g < 0.f ? 0.f : g;   // (a NaN stays)
  if (GRAD) d = g > 0.f ? 1.f : 0.f;
}
// a = act(g), d = act'(g) of eight; one branch for all of them
template <bool GRAD>
__device__ __forceinline__ void activate8(int act, const float* g, float* a, float* d) {
  if (act == kActSilu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) act_silu<GRAD>(g[e], a[e], d[e]);
  } else if (act == kActGelu) {
#pragma unroll 1
    for (int e = 0; e < 8; e += 4) {   // (erf is long)
      float x[4], y[4], z[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = e ? g[4 + i] : g[i];
        act_gelu<GRAD>(x[i], y[i], z[i]);
        (e ? a[4 + i] : a[i]) = y[i];
        if (GRAD) (e ? d[4 + i] : d[i]) = z[i];
      }
    }
  } else if (act == kActGeluTanh) {
#pragma unroll
    for (int e = 0; e < 8; ++e) act_gelu_tanh<GRAD>(g[e], a[e], d[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) act_relu<GRAD>(g[e], a[e], d[e]);
  }
}

// ------------------------------------------------------------------------------------------------------------- elements
template <typename T>
struct TileType;
template <>
struct TileType<bf16_t> {
  static constexpr int kPiece = 8, kStep = 64;    // elements of 16 bytes; k of a step
  static __device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
    return mfma16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  }
};
template <>
struct TileType<float> {
  static constexpr int kPiece = 4, kStep = 32;
  // each of the four instructions takes one k from each of the four lane groups' pieces
  static __device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// eight neighbouring numbers of C
__device__ __forceinline__ void tile_store8(bf16_t* p, const float* x) {
  const bf16x2 a = pack2(x[0], x[1]), b = pack2(x[2], x[3]), c = pack2(x[4], x[5]), d = pack2(x[6], x[7]);
  *(bf16x8*)p = bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ void tile_store8(float* p, const float* x) {
  *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
  *(f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void tile_load8(const bf16_t* p, float* x) {
  const bf16x8 v = *(const bf16x8*)p;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}
__device__ __forceinline__ void tile_load8(const float* p, float* x) {
  const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e < 4 ? lo[e & 3] : hi[e & 3];
}

// eight neighbouring numbers as they are kept, from fp32 and back
template <typename T>
struct Kept8;
template <>
struct Kept8<float> {
  f32x4 lo, hi;
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    lo = *(const f32x4*)((const float*)p + at);
    hi = *(const f32x4*)((const float*)p + at + 4);
  }
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < 4 ? lo[e & 3] : hi[e & 3];
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float* x) { tile_store8((float*)p + at, x); }
};
// Of bf16 rows: fp16 numbers, less their lowest bits, times a power of two that eight share, whose eight bits stand in those: the largest of the
// eight is put just below 2^15.  An error of at most 2^-10 of a number, down to 2^-29 of the largest (there 2^-38 of it), where bf16 would have
// up to 2^-8: those alone would be as large in the gradients as all the other roundings together.  Zero and the sign stay what they are (the derivative
// at 0).  Eight with an infinity or a NaN among them are kept as the upper 15 bits of the fp32 numbers.
template <>
struct Kept8<bf16_t> {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  u32x4 w;
  __device__ __forceinline__ void load(const void* p, int64_t at) { w = *(const u32x4*)((const uint16_t*)p + at); }
  __device__ __forceinline__ void get(float* x) const {
    // the lowest bits of numbers 2 i and 2 i + 1 are bits i and 4 + i of the power
    const unsigned b = (w[0] & 0x10001u) | (w[1] & 0x10001u) << 1 | (w[2] & 0x10001u) << 2 | (w[3] & 0x10001u) << 3;
    const int code = (b | b >> 12) & 0xff;
    if (code == 255) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = __builtin_bit_cast(float, e & 1 ? w[e >> 1] & 0xfffe0000u : (w[e >> 1] & 0xfffeu) << 16);
    } else {
      const float unit = __builtin_ldexpf(1.f, code - 141);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)__builtin_bit_cast(f16x2, w[e >> 1] & 0xfffefffeu)[e & 1] * unit;
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float* x) {
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __builtin_bit_cast(unsigned, x[e]) << 1);   // (a NaN is above an infinity)
    const int code = max((int)(most >> 24), 1);    // the largest is below 2^(code - 126)
    u32x4 w;
    if (code == 255) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned a = __builtin_bit_cast(unsigned, x[2 * i]), b = __builtin_bit_cast(unsigned, x[2 * i + 1]);
        if (x[2 * i] != x[2 * i]) a |= 0x20000u;    // (a NaN whose upper bits are an infinity's)
        if (x[2 * i + 1] != x[2 * i + 1]) b |= 0x20000u;
        w[i] = a >> 16 | (b & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)   // cut off at the lowest bit, and rounded at the one above it, away from zero halfway
        w[i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(__builtin_ldexpf(x[2 * i], 141 - code), __builtin_ldexpf(x[2 * i + 1], 141 - code))) + 0x10001u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (w[i] & 0xfffefffeu) | (code >> i & 1) | (code >> (4 + i) & 1) << 16;
    *(u32x4*)((uint16_t*)p + at) = w;
  }
};
// dg and du of eight numbers of the gradient of h
template <typename T>
__device__ __forceinline__ void gated_grad8(int act, const float* dh, const Kept8<T>& gate, const Kept8<T>& up, float* dg, float* du) {
  float g[8], u[8];
  gate.get(g);
  up.get(u);
  float a[8], d[8];
  activate8<true>(act, g, a, d);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    dg[e] = dh[e] * u[e] * d[e];
    du[e] = dh[e] * a[e];
  }
}

// row of a wave's part of an operand that entry j of fragment f stands for; PAIRS: two fragments share 32 rows (see above)
template <bool PAIRS>
__device__ __forceinline__ constexpr int frag_row(int f, int j) {
  return PAIRS ? 32 * (f >> 1) + 8 * (j >> 2) + 4 * (f & 1) + (j & 3) : 16 * f + j;
}

// a value that is the same in all lanes, in scalar registers whatever computed it (a division is done in vector registers, and a buffer's
// description from there would be walked lane by lane)
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t scalar64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)scalar((int)x) | (uint64_t)(uint32_t)scalar((int)(x >> 32)) << 32);
}

constexpr uint32_t kBeyond = 0x80000000u;   // an offset that no buffer's bounds reach

// ------------------------------------------------------------------------------------------------------- an operand's way
// ROWS rows of a step, loaded by WAVES waves, read in NF fragments by a wave whose part begins at row `base`; HALVES: every other 32 rows
// come from the second matrix.
template <typename T, bool COLS, int ROWS, int WAVES, int NF, bool PAIRS, bool HALVES>
struct OperandWay {
  typedef TileType<T> E;
  static constexpr int kBytes = ROWS * 128;
  static constexpr int kLoads = kBytes / 1024 / WAVES;                   // of a wave: 64 lanes of 16 bytes
  static constexpr int kLine = COLS ? ROWS * (int)sizeof(T) : 128;        // bytes of a row or a k
  static_assert(kBytes % (1024 * WAVES) == 0 && (!COLS || kLine >= 256) && (!COLS || (!PAIRS && (kLine % 256 == 0 || kLine == 384))), "tile");

  // Lanes 0-3, 12-15, 20-23 and 24-27 of a 16-byte read meet in the banks, and so do the other half of 32 lanes; of an 8-byte transposing
  // read all 32.  (Taken as sixteen neighbours, the reads of a step were 8 cycles each instead of 4.)
  static __device__ __forceinline__ int swizzle(int line) {
    if constexpr (!COLS) {
      const int q = (PAIRS ? line >> 3 : line >> 2) & 3;
      return (q >> 1) | ((q ^ (q >> 1)) & 1) << 1 | (line & 2) << 1;
    } else if constexpr (sizeof(T) == 2) {
      if constexpr (kLine % 256) return (line & 2) | ((line >> 3) & 1) << 2;   // (192 rows: every second line begins in the other half of the banks)
      else return 2 * ((line & 3) | ((line >> 3) & 1) << 2);
    } else {
      return 4 * ((line >> 2) & 3);
    }
  }

  uint32_t off[kLoads];   // of a lane's pieces from the step's beginning
  int piece;              // rows: the piece's number in the step is this, changed by the swizzle of the load's first line
  const char* at;         // the step's beginning
  int64_t left;           // bytes from there to the end of the matrix
  int64_t advance;

  __device__ __forceinline__ void begin(int64_t ld, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int instr = wave * kLoads + j, p = instr * 64 + lane;
      const int line = p / (kLine / 16), pc = (p % (kLine / 16)) ^ swizzle(line);
      int row = line;
      if constexpr (HALVES) {
        static_assert(!HALVES || (!COLS && kLoads == 4), "a wave's loads are of 32 rows, all of one matrix");
        row = 32 * (line >> 6) + (line & 31);
      }
      off[j] = (uint32_t)(row * ld) + pc * 16;
    }
    piece = (lane & 7) ^ swizzle(lane >> 3);
    advance = COLS ? E::kStep * ld : 128;
  }
  __device__ __forceinline__ void place(const TileOperand& o, const char* p, int row0, int k0, int k) {
    const int64_t to = COLS ? k0 * o.ld + row0 * (int64_t)sizeof(T) : row0 * o.ld + k0 * (int64_t)sizeof(T);
    const int64_t end = COLS ? (k - 1) * o.ld + o.rows * (int64_t)sizeof(T) : (o.rows - 1) * o.ld + k * (int64_t)sizeof(T);
    at = (const char*)scalar64((int64_t)(p + to));
    left = scalar64(end - to);
  }
  // loads of a step into its place in LDS; k_left: numbers of k from the step's beginning on
  __device__ __forceinline__ void load(char* lds, int wave, int k_left) {
    const int bound = left <= 0 ? 0 : left > (int64_t)kBeyond ? (int)kBeyond : (int)left;
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, bound, 0x00027000);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int instr = wave * kLoads + j;
      uint32_t o = off[j];
      if constexpr (!COLS) o = (piece ^ swizzle(8 * instr)) * E::kPiece < k_left ? o : kBeyond;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + instr * 1024), 16, o, 0, 0, 0);
    }
    at += advance;
    left -= advance;
  }
  static constexpr int kReads = NF * (!COLS ? 1 : sizeof(T) == 2 ? 2 : 4);   // of half a step, by a wave

  // places of a lane's fragments in a step
  static constexpr int kPlaces = !COLS ? 2 : NF;
  uint32_t place_of[kPlaces];
  __device__ __forceinline__ void aim(int base, int lane) {
    const int j = lane & 15, g = lane >> 4;
    if constexpr (!COLS) {
      const int row = base + frag_row<PAIRS>(0, j);
#pragma unroll
      for (int h = 0; h < 2; ++h) place_of[h] = row * 128 + (((4 * h + g) ^ swizzle(row)) * 16);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int f = 0; f < kPlaces; ++f) {
        const int k = 8 * g + (j >> 2), col = base + 16 * f + 4 * (j & 3);
        place_of[f] = k * kLine + (((col >> 3) ^ swizzle(k)) * 16) + (col & 7) * 2;
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int k = 4 * g, col = base + frag_row<PAIRS>(f, j);
        place_of[f] = k * kLine + (((col >> 2) ^ swizzle(k)) * 16) + (col & 3) * 4;
      }
    }
  }
  __device__ __forceinline__ f32x4 read(const char* step, int half, int f) const {
    if constexpr (!COLS) {
      return *(const f32x4*)(step + place_of[half] + frag_row<PAIRS>(f, 0) * 128);
    } else {
      const char* p = step + half * (E::kStep / 2) * kLine;
      if constexpr (sizeof(T) == 2) {
        p += place_of[f];
        return __builtin_bit_cast(f32x4, join(lds_read_tr((const bf16_t*)p), lds_read_tr((const bf16_t*)(p + 4 * kLine))));
      } else {
        p += place_of[f];
        return f32x4{*(const float*)p, *(const float*)(p + kLine), *(const float*)(p + 2 * kLine), *(const float*)(p + 3 * kLine)};
      }
    }
  }
};

template <int N>
__device__ __forceinline__ void wait_loads_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// WM x WN waves, each with NFM x NFN fragments of 16 x 16
template <typename T, int KIND, bool ACOLS, bool BCOLS, int WM, int WN, int NFM, int NFN>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_product_kernel(TileArgs P) {
  typedef TileType<T> E;
  constexpr int W = WM * WN, BM = 16 * NFM * WM, BN = 16 * NFN * WN;
  typedef OperandWay<T, ACOLS, BM, W, NFM, false, false> AWay;
  typedef OperandWay<T, BCOLS, BN, W, NFN, !BCOLS, KIND == kTileGated> BWay;
  constexpr uint32_t kStepBytes = AWay::kBytes + BWay::kBytes;
  constexpr int kLoads = AWay::kLoads + BWay::kLoads;
  extern __shared__ __attribute__((aligned(16))) char ring[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

  // Tiles in order go to the dies in eight runs, so that a die's cache holds the operands of neighbours; the workgroups of a die take
  // its run's tiles in turn.
  const int all = P.tiles * P.splits, die = blockIdx.x & 7;
  const int run = (all >> 3) + (die < (all & 7)), run0 = die * (all >> 3) + min(die, all & 7);
  const int takers = (gridDim.x >> 3) + (die < (int)(gridDim.x & 7)), mine = blockIdx.x >> 3;
  const int one = (P.k + E::kStep - 1) / E::kStep;         // steps of a matrix
  constexpr int kCols = KIND == kTileGated ? BN / 2 : BN;
  struct Place { int which, m0, n0, split, step, end; };
  auto where = [&](int i) {
    Place w;
    const int place = run0 + i;
    w.split = place / P.tiles;
    const int tile = place - w.split * P.tiles;
    w.which = 0;
    if (P.n_prod > 1 && tile >= P.prod[1].first) w.which = 1;
    if (P.n_prod > 2 && tile >= P.prod[2].first) w.which = 2;
    const TileProduct& pr = P.prod[w.which];
    // bands of eight tiles of m, in a band down the tiles of m first
    const int tiles_m = (pr.a.rows + BM - 1) / BM, in = tile - pr.first, band = in / (8 * pr.tiles_n), in_band = in - band * 8 * pr.tiles_n;
    const int high = min(8, tiles_m - 8 * band), tn = in_band / high, tm = 8 * band + in_band - tn * high;
    w.m0 = scalar(tm * BM);
    w.n0 = scalar(tn * kCols);
    w.split = scalar(w.split);
    w.which = scalar(w.which);
    w.step = w.split * P.split_steps;
    w.end = min(KIND == kTileTwice ? 2 * one : one, w.step + P.split_steps);
    return w;
  };

  // Loads run two steps ahead of the products, over the ends of matrices and tiles: the next tile's first steps are on their way while
  // this one's results are stored.
  AWay A;
  BWay B;
  int ahead = mine, which = -1, to_go = 0, k_left = 0;     // the tile that is loaded; steps left of its present matrix
  uint32_t slot = 0;
  Place next{};
  auto second_of = [&](int w) { return KIND == kTileTwice && w >= one; };
  auto go_on = [&]() {                                     // to the next matrix, the next tile, or nowhere
    if (to_go) return;
    if (next.step >= next.end) {
      if (ahead >= run) {
        A.left = B.left = 0;
        k_left = 0;
        to_go = -1;
        return;
      }
      next = where(ahead);
      ahead += takers;
    }
    const TileProduct& pr = P.prod[next.which];
    if (next.which != which) {
      which = next.which;
      A.begin(pr.a.ld, wave, lane);
      B.begin(pr.b.ld, wave, lane);
    }
    const bool second = second_of(next.step);
    const int k0 = (second ? next.step - one : next.step) * E::kStep, end = KIND == kTileTwice && !second ? min(one, next.end) : next.end;
    A.place(pr.a, second ? pr.a.p2 : pr.a.p, next.m0, k0, P.k);
    B.place(pr.b, (KIND == kTileGated ? (wave & 1) != 0 : second) ? pr.b.p2 : pr.b.p, next.n0, k0, P.k);
    k_left = P.k - k0;
    to_go = end - next.step;
    next.step = end;
  };
  auto issue = [&](uint32_t to) {
    A.load(ring + to, wave, k_left);
    B.load(ring + to + AWay::kBytes, wave, k_left);
    k_left -= E::kStep;
    --to_go;
  };
  A.aim(wave / WN * 16 * NFM, lane);
  B.aim(wave % WN * 16 * NFN, lane);
  go_on();
  issue(0);
  go_on();
  issue(kStepBytes);
  go_on();

  f32x4 acc[NFM][NFN];
  // A step in four parts: the half of k by the half of a wave's rows of A.  Operands of a part are read during the one before.
  constexpr int HM = NFM / 2;
  f32x4 a_low[HM], a_high[HM], b_first[NFN], b_second[NFN];
  auto read_a = [&](f32x4 (&f)[HM], uint32_t at, int half, int m0) {
#pragma unroll
    for (int m = 0; m < HM; ++m) f[m] = A.read(ring + at, half, m0 + m);
  };
  auto read_b = [&](f32x4 (&f)[NFN], uint32_t at, int half) {
#pragma unroll
    for (int n = 0; n < NFN; ++n) f[n] = B.read(ring + at + AWay::kBytes, half, n);
  };
  auto multiply = [&](const f32x4 (&a)[HM], const f32x4 (&b)[NFN], int m0) {
#pragma unroll
    for (int m = 0; m < HM; ++m)
#pragma unroll
      for (int n = 0; n < NFN; ++n) acc[m0 + m][n] = E::mma(b[n], a[m], acc[m0 + m][n]);
  };
  // the matrix units are fed without a pause: reads, then loads go out between their instructions
  auto spread = [&](auto reads, auto loads) {
    constexpr int kR = decltype(reads)::value, kL = decltype(loads)::value, kMma = HM * NFN * (sizeof(T) == 2 ? 1 : 4);
    constexpr int kEach = kMma / (kR + kL) > 0 ? kMma / (kR + kL) : 1;
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    }
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  typedef std::integral_constant<int, 0> None;
  typedef std::integral_constant<int, AWay::kReads / 2> ReadsA;
  typedef std::integral_constant<int, AWay::kReads / 2 + BWay::kReads> ReadsAB;
  typedef std::integral_constant<int, kLoads> Loads;

  // a lane: row j of fragment m, columns 8 g .. of a pair of fragments n
  auto store_tile = [&](const TileProduct& pr, const Place& at_tile) {
    const int M = pr.a.rows, N = pr.b.rows, split = at_tile.split;
    if constexpr (BCOLS) {
      asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");   // the last products' results, which the compiler does not see the swaps read
#pragma unroll
      for (int m = 0; m < NFM; ++m)
#pragma unroll
        for (int n = 0; n < NFN; n += 2)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a = acc[m][n][e], b = acc[m][n + 1][e];
            swap_halves(a, b);
            swap_rows(a, b);
            acc[m][n][e] = a;
            acc[m][n + 1][e] = b;
          }
    }
    const int j = lane & 15, g = lane >> 4, m0 = at_tile.m0 + wave / WN * 16 * NFM;
    const int n0 = at_tile.n0 + wave % WN * (kCols / WN) + 8 * g;
    if constexpr (KIND == kTileGated || KIND == kTileGrad) {
      // Columns of padding are zero whatever the product is: the weights are zero there, but beside an infinity in a row of x or dy it is a NaN, which
      // the next product, over these columns, would spread over the whole row.
      if (P.used < N && at_tile.n0 + kCols > P.used) {
#pragma unroll
        for (int n = 0; n < NFN; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool own = n0 + (KIND == kTileGated ? 0 : 32 * (n >> 1)) + 4 * (n & 1) + e < P.used;
#pragma unroll
            for (int m = 0; m < NFM; ++m) acc[m][n][e] = own ? acc[m][n][e] : 0.f;
          }
      }
    }
    if constexpr (KIND == kTileGrad) {
      if (P.splits == 1) {
        // The factors are on their way kAhead fragments ahead of their use: a wait for them is one for the stores that went out before them.
        constexpr int kAhead = sizeof(T) == 2 ? 2 : 1;
        Kept8<T> gate[kAhead + 1][NFN / 2], up[kAhead + 1][NFN / 2];
        auto fetch = [&](int m) {
          const int row = min(m0 + frag_row<false>(m, j), M - 1);
#pragma unroll
          for (int n = 0; n < NFN / 2; ++n) {
            const int64_t at = row * pr.ldc + min(n0 + 32 * n, N - 8);
            gate[m % (kAhead + 1)][n].load(P.kept.gate, at);
            up[m % (kAhead + 1)][n].load(P.kept.up, at);
          }
        };
#pragma unroll
        for (int m = 0; m < kAhead && m < NFM; ++m) fetch(m);
#pragma unroll
        for (int m = 0; m < NFM; ++m) {
          if (m + kAhead < NFM) fetch(m + kAhead);
          const int row = m0 + frag_row<false>(m, j);
#pragma unroll
          for (int n = 0; n < NFN / 2; ++n) {
            float c[8], dg[8], du[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = acc[m][2 * n + (e >> 2)][e & 3];
            gated_grad8(P.act, c, gate[m % (kAhead + 1)][n], up[m % (kAhead + 1)][n], dg, du);
            if (row < M && n0 + 32 * n < N) {
              const int64_t at = row * pr.ldc + n0 + 32 * n;
              tile_store8((T*)pr.c + at, dg);
              tile_store8((T*)P.c2 + at, du);
            }
          }
        }
        return;
      }
    }
#pragma unroll
    for (int m = 0; m < NFM; ++m) {
      const int row = m0 + frag_row<false>(m, j);
      if (row >= M) continue;
      if constexpr (KIND == kTileGated) {
        static_assert(KIND != kTileGated || NFN == 4, "a wave has 32 columns of each matrix");
        if (n0 >= N) continue;
        float gt[8], up[8], c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gt[e] = acc[m][e >> 2][e & 3];
          up[e] = acc[m][2 + (e >> 2)][e & 3];
        }
        if (P.splits > 1) {
          float* part = pr.part + ((int64_t)split * M + row) * (2 * (int64_t)N) + n0;
          tile_store8(part, gt);
          tile_store8(part + N, up);
          continue;
        }
        activate8<false>(P.act, gt, c, nullptr);
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] *= up[e];
        const int64_t at = row * pr.ldc + n0;
        tile_store8((T*)pr.c + at, c);
        if (P.kept.gate) {
          Kept8<T>::store(P.kept.gate, at, gt);
          Kept8<T>::store(P.kept.up, at, up);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NFN / 2; ++n) {
          const int col = n0 + 32 * n;
          if (col >= N) continue;
          float c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = acc[m][2 * n + (e >> 2)][e & 3];
          if (P.splits > 1) tile_store8(pr.part + ((int64_t)split * M + row) * N + col, c);
          else tile_store8((T*)pr.c + row * pr.ldc + col, c);
        }
      }
    }
  };
  wait_loads_and_meet<kLoads>();
  read_b(b_first, 0, 0);
  read_a(a_low, 0, 0, 0);
  for (int tile = mine; tile < run; tile += takers) {
    const Place at = where(tile);
    const TileProduct& pr = P.prod[at.which];
#pragma unroll
    for (int m = 0; m < NFM; ++m)
#pragma unroll
      for (int n = 0; n < NFN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = at.step; s < at.end; ++s) {
      read_a(a_high, slot, 0, HM);
      multiply(a_low, b_first, 0);
      spread(ReadsA(), None());
      read_b(b_second, slot, 1);
      read_a(a_low, slot, 1, 0);
      multiply(a_high, b_first, HM);
      spread(ReadsAB(), None());
      read_a(a_high, slot, 1, HM);
      multiply(a_low, b_second, 0);
      spread(ReadsA(), None());
      wait_loads_and_meet<0>();
      __builtin_amdgcn_sched_barrier(0);
      read_b(b_first, slot ^ kStepBytes, 0);
      read_a(a_low, slot ^ kStepBytes, 0, 0);
      issue(slot);
      multiply(a_high, b_second, HM);
      spread(ReadsAB(), Loads());
      slot ^= kStepBytes;
      go_on();
    }
    store_tile(pr, at);
    if constexpr (KIND == kTileGrad) {                   // (its registers are needed there: the operands are read again)
      read_b(b_first, slot, 0);
      read_a(a_low, slot, 0, 0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // loads into LDS do not outlive the workgroup
}

}  // namespace pal
