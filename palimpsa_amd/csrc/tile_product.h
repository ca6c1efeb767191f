// Products of two matrices on the matrix units, tile by tile:  C[m][n] = sum_k A(m, k) B(n, k),  rows of bf16 or fp32, sums in fp32.
//
// Either operand lies with its k side by side ("rows": element (i, k) at i ld + k) or its rows side by side ("columns": at k ld + i), so that the
// products of a layer's forward pass (rows, rows), of the gradient of its input (rows, columns) and of its weight (columns, columns) all
// read their operands as they lie in memory.
//
// A workgroup takes a tile of BM x BN.  64 bytes of k of both operands (32 bf16 or 16 fp32 numbers) are a step; a ring of four steps is
// kept in LDS, filled by loads that write LDS directly (no registers, three steps ahead), and each wave reads its operands of the next
// step into a second set of registers while the matrix units work on the present one.  A step needs one barrier: behind it the loads of the
// next step have landed for all waves, and the present step's place in the ring, which all have read, is free.
//
// Layout of a step in LDS: pieces of 16 bytes, a row of an operand that lies in rows as four pieces, a k of one that lies in columns as
// BM / 8 (BM / 4) pieces, in either case with the piece's number changed by an exclusive or (`swizzle`) so that the sixteen lanes that
// read at one time find sixteen different places among the banks.  (The direct loads write lane after lane, so the change is made to the
// address that a lane reads from.)
//
// The 16 x 16 results are arranged so that a lane holds eight neighbouring columns of C of one row: matrix instruction (n, m) takes rows
// 32 (f / 2) + 8 (j / 4) + 4 (f % 2) + j % 4, j < 16, of a wave's part of either operand as its fragment f, and B stands first, so that its index
// runs along a lane's four numbers.  Two fragments together are 16-byte stores without a turn through LDS.
//
// Whatever lies behind a matrix (rows behind the last one, k behind the end) is read as zero: by the bounds of the buffer for whole rows,
// by an address beyond all bounds for the rest of a row.
#pragma once
#include "pal_common.h"

namespace pal {

struct TileOperand {
  const char* p;       // element (0, 0)
  const char* p2;      // second matrix of the same shape (NULL: none): see TileArgs
  int64_t ld;          // bytes from row to row (lies in rows) or from k to k (lies in columns)
  int32_t rows;        // m or n
};

// up to three products over the same k in one launch
struct TileProduct {
  TileOperand a, b;
  void* c;             // [m][n], packed
  float* part;         // [splits][m][n] where k is split
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
  // for the feed-forward block's kinds: rows [m][n] beside C
  const void *gate, *up;
  void *gate_out, *up_out;
  int32_t act;
};

enum TileKind {
  kTilePlain = 0,
  kTileGated,   // b has two matrices, half of a tile's columns from each: C = act(A B^T) (A B2^T), both factors kept beside it if asked
  kTileGrad,    // D = A B^T is the gradient of such a C: from its factors the gradients of both (c, up_out) and C itself (gate_out)
  kTileTwice,   // A B^T + A2 B2^T
};

// ---------------------------------------------------------------------------------------------------------- activations
enum { kActSilu = PAL_ACT_SILU, kActGelu = PAL_ACT_GELU, kActGeluTanh = PAL_ACT_GELU_TANH, kActRelu = PAL_ACT_RELU };

__device__ __forceinline__ float act_logistic(float x) { return fast_rcp(1.f + __expf(-x)); }
// a = act(g), d = act'(g)
template <bool GRAD>
__device__ __forceinline__ void activate(int act, float g, float& a, float& d) {
  if (act == kActSilu) {
    const float f = act_logistic(g);
    a = g * f;
    if (GRAD) d = f * fmaf(g, 1.f - f, 1.f);
  } else if (act == kActGelu) {
    const float f = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * f;
    if (GRAD) d = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), f);
  } else if (act == kActGeluTanh) {
    // (1 + tanh(z / 2)) / 2 is the logistic function of z
    const float g2 = g * g, f = act_logistic(1.5957691216057308f * g * fmaf(0.044715f, g2, 1.f));
    a = g * f;
    if (GRAD) {
      const float s = f * (1.f - f);
      d = s > 0.f ? fmaf(1.5957691216057308f * g * s, fmaf(0.134145f, g2, 1.f), f) : f;   // (no 0 times infinity far out)
    }
  } else {
    a = g < 0.f ? 0.f : g;   // (a NaN stays)
    if (GRAD) d = g > 0.f ? 1.f : 0.f;
  }
}

// ------------------------------------------------------------------------------------------------------------- elements
template <typename T>
struct TileType;
template <>
struct TileType<bf16_t> {
  static constexpr int kPiece = 8, kStep = 32;    // elements of 16 bytes; k of a step
  static __device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
    return mfma16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  }
};
template <>
struct TileType<float> {
  static constexpr int kPiece = 4, kStep = 16;
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

// row of a wave's part of an operand that entry j of fragment f stands for
__device__ __forceinline__ constexpr int frag_row(int f, int j) { return 32 * (f >> 1) + 8 * (j >> 2) + 4 * (f & 1) + (j & 3); }

constexpr uint32_t kBeyond = 0x80000000u;   // an offset that no buffer's bounds reach
constexpr int kRing = 4;

// ------------------------------------------------------------------------------------------------------- an operand's way
// ROWS rows of a step, loaded by WAVES waves, read in NF fragments by a wave whose part begins at row `base`; HALVES: every other 32 rows
// come from the second matrix.
template <typename T, bool COLS, int ROWS, int WAVES, int NF, bool HALVES>
struct OperandWay {
  typedef TileType<T> E;
  static constexpr int kBytes = ROWS * 64;
  static constexpr int kLoads = kBytes / 1024 / WAVES;                   // of a wave: 64 lanes of 16 bytes
  static constexpr int kLine = COLS ? ROWS * (int)sizeof(T) : 64;         // bytes of a row or a k
  static_assert(kBytes % (1024 * WAVES) == 0 && (!COLS || kLine >= 256), "tile");

  static __device__ __forceinline__ int swizzle(int line) {
    if constexpr (!COLS) return (line >> 3) & 3;
    else if constexpr (sizeof(T) == 2) return 4 * (line & 3);
    else return ((line >> 2) & 1) | ((line & 8));
  }

  uint32_t off[kLoads];   // of a lane's pieces from the step's beginning
  int kpos[kLoads];       // rows: the piece's k in the step
  const char* at;         // the step's beginning
  int64_t left;           // bytes from there to the end of the matrix
  int64_t advance;

  __device__ __forceinline__ void begin(const TileOperand& o, int row0, int k0, int k, int wave, int lane) {
    bool second = false;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int instr = wave * kLoads + j, p = instr * 64 + lane;
      const int line = p / (kLine / 16), piece = (p % (kLine / 16)) ^ swizzle(line);
      if constexpr (COLS) {
        off[j] = (uint32_t)(line * o.ld) + piece * 16;
        kpos[j] = 0;
      } else {
        int row = line;
        if constexpr (HALVES) {
          static_assert(!HALVES || kLoads == 2, "a wave's loads are of one matrix");
          second = wave & 1;
          row = 32 * (line >> 6) + (line & 31);
        }
        off[j] = (uint32_t)(row * o.ld) + piece * 16;
        kpos[j] = piece * E::kPiece;
      }
    }
    const char* p = second ? o.p2 : o.p;
    place(o, p, row0, k0, k);
    advance = COLS ? E::kStep * o.ld : 64;
  }
  __device__ __forceinline__ void place(const TileOperand& o, const char* p, int row0, int k0, int k) {
    const int64_t to = COLS ? k0 * o.ld + row0 * (int64_t)sizeof(T) : row0 * o.ld + k0 * (int64_t)sizeof(T);
    const int64_t end = COLS ? (k - 1) * o.ld + o.rows * (int64_t)sizeof(T) : (o.rows - 1) * o.ld + k * (int64_t)sizeof(T);
    at = p + to;
    left = end - to;
  }
  // loads of a step into its place in LDS; k_left: numbers of k from the step's beginning on
  __device__ __forceinline__ void load(char* lds, int wave, int k_left) {
    const int bound = left <= 0 ? 0 : left > (int64_t)kBeyond ? (int)kBeyond : (int)left;
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, bound, 0x00027000);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      uint32_t o = off[j];
      if constexpr (!COLS) o = kpos[j] < k_left ? o : kBeyond;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + (wave * kLoads + j) * 1024), 16, o, 0, 0, 0);
    }
    at += advance;
    left -= advance;
  }

  // places of a lane's fragments in a step
  static constexpr int kPlaces = !COLS ? 1 : sizeof(T) == 2 ? NF / 2 : NF;
  uint32_t place_of[kPlaces];
  __device__ __forceinline__ void aim(int base, int lane) {
    const int j = lane & 15, g = lane >> 4;
    if constexpr (!COLS) {
      const int row = base + frag_row(0, j);
      place_of[0] = row * 64 + ((g ^ swizzle(row)) * 16);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int f = 0; f < NF / 2; ++f) {
        const int k = 8 * g + (j >> 2), col = base + 32 * f + 8 * (j & 3);
        place_of[f] = k * kLine + (((col >> 3) ^ swizzle(k)) * 16);
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int k = 4 * g, col = base + frag_row(f, j);
        place_of[f] = k * kLine + (((col >> 2) ^ swizzle(k)) * 16) + (col & 3) * 4;
      }
    }
  }
  __device__ __forceinline__ f32x4 read(const char* step, int f) const {
    if constexpr (!COLS) {
      return *(const f32x4*)(step + place_of[0] + (32 * (f >> 1) + 4 * (f & 1)) * 64);
    } else if constexpr (sizeof(T) == 2) {
      const char* p = step + place_of[f >> 1] + 8 * (f & 1);
      return __builtin_bit_cast(f32x4, join(lds_read_tr((const bf16_t*)p), lds_read_tr((const bf16_t*)(p + 4 * kLine))));
    } else {
      const char* p = step + place_of[f];
      return f32x4{*(const float*)p, *(const float*)(p + kLine), *(const float*)(p + 2 * kLine), *(const float*)(p + 3 * kLine)};
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
  typedef OperandWay<T, ACOLS, BM, W, NFM, false> AWay;
  typedef OperandWay<T, BCOLS, BN, W, NFN, KIND == kTileGated> BWay;
  constexpr int kStepBytes = AWay::kBytes + BWay::kBytes, kLoads = AWay::kLoads + BWay::kLoads;
  extern __shared__ __attribute__((aligned(16))) char ring[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

  // tiles in order go to one die after the other: each gets a run of neighbouring ones, whose operands its cache then holds
  const int all = P.tiles * P.splits, id = blockIdx.x, die = id & 7, q = all >> 3, r = all & 7;
  const int place = die * q + min(die, r) + (id >> 3);
  const int split = place / P.tiles, tile = place - split * P.tiles;
  int which = 0;
  if (P.n_prod > 1 && tile >= P.prod[1].first) which = 1;
  if (P.n_prod > 2 && tile >= P.prod[2].first) which = 2;
  const TileProduct& pr = P.prod[which];
  const int M = pr.a.rows, N = pr.b.rows, tiles_m = (M + BM - 1) / BM;
  // bands of eight tiles of m, in a band down the tiles of m first
  const int in = tile - pr.first, band = in / (8 * pr.tiles_n), in_band = in - band * 8 * pr.tiles_n;
  const int high = min(8, tiles_m - 8 * band), tn = in_band / high, tm = 8 * band + in_band - tn * high;
  constexpr int kCols = KIND == kTileGated ? BN / 2 : BN;
  const int m0 = tm * BM, n0 = tn * kCols;

  int step = split * P.split_steps;
  const int one = (P.k + E::kStep - 1) / E::kStep;         // steps of a matrix
  const int end = min(KIND == kTileTwice ? 2 * one : one, step + P.split_steps);
  const int steps = end - step;
  AWay A;
  BWay B;
  int k_left, to_second = 0;                                // steps until the second matrix
  {
    const bool second = KIND == kTileTwice && step >= one;
    const int k0 = (second ? step - one : step) * E::kStep;
    TileOperand oa = pr.a, ob = pr.b;
    if (second) oa.p = oa.p2, ob.p = ob.p2;
    A.begin(oa, m0, k0, P.k, wave, lane);
    B.begin(ob, n0, k0, P.k, wave, lane);
    k_left = P.k - k0;
    if (KIND == kTileTwice) to_second = second ? -1 : one - step;
  }
  A.aim(wave / WN * 16 * NFM, lane);
  B.aim(wave % WN * 16 * NFN, lane);

  int issued = 0;
  auto issue = [&]() {
    char* to = ring + (issued & (kRing - 1)) * kStepBytes;
    const int k = issued < steps ? k_left : 0;
    if (issued >= steps) A.left = 0, B.left = 0;            // nothing is read; the counts of loads in flight stay the same
    A.load(to, wave, k);
    B.load(to + AWay::kBytes, wave, k);
    k_left -= E::kStep;
    ++issued;
    if (KIND == kTileTwice && issued == to_second) {
      A.place(pr.a, pr.a.p2, m0, 0, P.k);
      B.place(pr.b, pr.b.p2, n0, 0, P.k);
      k_left = P.k;
    }
  };
#pragma unroll
  for (int s = 0; s < kRing; ++s) issue();

  f32x4 acc[NFM][NFN];
#pragma unroll
  for (int m = 0; m < NFM; ++m)
#pragma unroll
    for (int n = 0; n < NFN; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Frags { f32x4 a[NFM], b[NFN]; } now, next;
  auto read = [&](Frags& f, int s) {
    const char* at = ring + (s & (kRing - 1)) * kStepBytes;
#pragma unroll
    for (int n = 0; n < NFN; ++n) f.b[n] = B.read(at + AWay::kBytes, n);
#pragma unroll
    for (int m = 0; m < NFM; ++m) f.a[m] = A.read(at, m);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int m = 0; m < NFM; ++m)
#pragma unroll
      for (int n = 0; n < NFN; ++n) acc[m][n] = E::mma(f.b[n], f.a[m], acc[m][n]);
  };
  wait_loads_and_meet<(kRing - 1) * kLoads>();
  read(now, 0);
  // a step: the loads of the next one have landed, this one's place is free
  auto turn = [&](Frags& f, Frags& g, int s) {
    wait_loads_and_meet<(kRing - 2) * kLoads>();
    issue();
    read(g, s + 1);
    multiply(f);
  };
  int s = 0;
  for (; s + 2 <= steps; s += 2) {
    turn(now, next, s);
    turn(next, now, s + 1);
  }
  if (s < steps) multiply(now);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // loads into LDS do not outlive the workgroup

  // a lane: row j of fragment m, columns 8 g .. of a pair of fragments n
  const int j = lane & 15, g = lane >> 4, mw = m0 + wave / WN * 16 * NFM;
#pragma unroll
  for (int m = 0; m < NFM; ++m) {
    const int row = mw + frag_row(m, j);
    if (row >= M) continue;
    if constexpr (KIND == kTileGated) {
#pragma unroll
      for (int n = 0; n < NFN; n += 4) {
        const int col = n0 + wave % WN * 8 * NFN + 8 * n + 8 * g;
        if (col >= N) continue;
        float gt[8], up[8], c[8], none;
#pragma unroll
        for (int e = 0; e < 8; ++e) gt[e] = acc[m][n + (e >> 2)][e & 3], up[e] = acc[m][n + 2 + (e >> 2)][e & 3];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          activate<false>(P.act, gt[e], c[e], none);
          c[e] *= up[e];
        }
        const int64_t at = (int64_t)row * N + col;
        tile_store8((T*)pr.c + at, c);
        if (P.gate_out) {
          tile_store8((T*)P.gate_out + at, gt);
          tile_store8((T*)P.up_out + at, up);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NFN; n += 2) {
        const int col = n0 + wave % WN * 16 * NFN + 16 * n + 8 * g;
        if (col >= N) continue;
        float c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = acc[m][n + (e >> 2)][e & 3];
        const int64_t at = (int64_t)row * N + col;
        if (P.splits > 1) {
          tile_store8(pr.part + (int64_t)split * M * N + at, c);
        } else if constexpr (KIND == kTileGrad) {
          float gt[8], up[8], dg[8], du[8], h[8];
          tile_load8((const T*)P.gate + at, gt);
          tile_load8((const T*)P.up + at, up);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a, d;
            activate<true>(P.act, gt[e], a, d);
            dg[e] = c[e] * up[e] * d;
            du[e] = c[e] * a;
            h[e] = a * up[e];
          }
          tile_store8((T*)pr.c + at, dg);
          tile_store8((T*)P.up_out + at, du);
          if (P.gate_out) tile_store8((T*)P.gate_out + at, h);
        } else {
          tile_store8((T*)pr.c + at, c);
        }
      }
    }
  }
}

}  // namespace pal
