// Gated feed-forward block:  g = x Wg^T,  u = x Wu^T,  h = act(g) u,  y = h Wd^T,  and its gradients
//     dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h.
//
// Forward: two launches.  The first computes both products of a tile side by side and stores h (for training g and u too); the second
// multiplies by Wd.  Backward: dh is never stored, the kernel that computes it turns it into dg and du; the gradient of x is one walk over
// both products, and the three of the weights are one launch (see tile_product.h).
//
// A call of few rows is bound by the weights: few_rows_kernel has no tiles in LDS, the waves of a workgroup walk over k side by side, weights and
// rows straight from memory into the matrix units.  Up to 16 rows, and up to 64 where the rows, which every workgroup reads, are not more traffic
// than small tiles with k in shares take (plan_few).
//
// Roundings to the type of the rows: h, dg and du, once each, half a step of the type, as operands of the matrix units; g and u are kept more
// exactly (Kept8); all sums are in fp32.  The errors in y and the gradients are then of the size of the rounding of those results themselves.  Up to
// sixteen rows of bf16 have h as a sum of two bf16 numbers, whose second product the weights' traffic hides (2048 -> 5632 -> 2048, one row: 20.7
// and 22.1 us; 32 rows, where it does not: 35.8 and 45.6).
#include "pal_common.h"
#include "pal_host.h"
#include "pal_profile.h"
#include "rows8.h"
#include "tile_product.h"

namespace pal {

constexpr int kFewRows = 64, kFewSpans = 4;

// ------------------------------------------------------------------------------------------------------------ few rows
struct FewArgs {
  const void *x, *w, *w2;    // [rows][k] (x_ld), [n][k]; w2: second product (gated)
  void* out;                 // [rows][n]
  Kept kept;
  int64_t x_ld, out_ld;      // elements
  int32_t rows, n, k, act;
  const void* x_low;         // bf16 rows of h: what its rounding left, to be added to x
  void* out_low;
  int32_t used;              // gated: see TileArgs
};

// R groups of sixteen rows of x.  The waves of a workgroup (as many as it has) take spans of 128 bytes of k in turn, four of them in one go (two of
// more groups of rows, whose registers leave a compute unit two workgroups then): 768 -> 2048 -> 768 of one row, replayed, 8.5 us where one at
// a time is 9.1, 2048 -> 5632 -> 2048 21.0 and 21.3.
template <typename T, bool GATED, int R>
__global__ __launch_bounds__(GATED ? 512 : 1024) void few_rows_kernel(FewArgs P) {
  typedef TileType<T> E;
  constexpr int B = R == 1 ? kFewSpans : kFewSpans / 2;
  constexpr bool kSplits = sizeof(T) == 2 && R == 1, kLow = kSplits && !GATED;   // h in two parts
  constexpr int kMats = GATED ? 2 : 1, kPiece = E::kPiece, kSpan = 8 * kPiece;
  extern __shared__ f32x4 shares[];                    // [waves][kMats * R][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int j = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const int64_t wrow = (int64_t)min(n0 + j, P.n - 1) * P.k;
  const T* w[2] = {(const T*)P.w + wrow, GATED ? (const T*)P.w2 + wrow : nullptr};
  const T *x[R], *x_low[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = min(16 * r + j, P.rows - 1) * P.x_ld;
    x[r] = (const T*)P.x + row;
    if constexpr (kLow) x_low[r] = (const T*)P.x_low + row;
  }
  f32x4 acc[kMats][R];
#pragma unroll
  for (int m = 0; m < kMats; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int turn = waves * kSpan;
  for (int k0 = wave * kSpan; k0 < P.k; k0 += B * turn) {
    // a span beyond the end is the last one once more, and counts as zero
    auto at = [&](int b, int h) { return min(k0 + b * turn + (4 * h + g) * kPiece, P.k - kPiece); };
    f32x4 wb[B][2][kMats], xb[B][2][R], xl[B][2][kLow ? R : 1];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          xb[b][h][r] = *(const f32x4*)(x[r] + at(b, h));
          if constexpr (kLow) xl[b][h][r] = *(const f32x4*)(x_low[r] + at(b, h));
        }
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < kMats; ++m) wb[b][h][m] = *(const f32x4*)(w[m] + at(b, h));
    __builtin_amdgcn_sched_barrier(0);                 // all of these are on their way before the first is waited for
#pragma unroll
    for (int b = 0; b < B; ++b) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = k0 + b * turn + (4 * h + g) * kPiece < P.k;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int m = 0; m < kMats; ++m) {
            acc[m][r] = E::mma(in ? wb[b][h][m] : zero, in ? xb[b][h][r] : zero, acc[m][r]);
            if constexpr (kLow) acc[m][r] = E::mma(in ? wb[b][h][m] : zero, in ? xl[b][h][r] : zero, acc[m][r]);
          }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kMats; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) shares[(wave * kMats * R + m * R + r) * 64 + lane] = acc[m][r];
  __syncthreads();
  // a thread: eight neighbouring columns of one row
  for (int i = threadIdx.x; i < R * 32; i += blockDim.x) {
    const int r = i >> 5, l = (i & 15) | (i & 16) << 1, row = 16 * r + (l & 15), n = n0 + 4 * (l >> 4);
    float t[kMats][8];
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
      f32x4 lo = zero, hi = zero;
#pragma unroll 4
      for (int v = 0; v < waves; ++v) {
        const f32x4* s = shares + (v * kMats * R + m * R + r) * 64 + l;
        lo += s[0];
        hi += s[16];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) t[m][e] = e < 4 ? lo[e & 3] : hi[e & 3];
    }
    if (row >= P.rows || n >= P.n) continue;
    const int64_t at = row * P.out_ld + n;
    if constexpr (GATED) {
      float c[8];
      if (n + 8 > P.used) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          t[0][e] = n + e < P.used ? t[0][e] : 0.f;
          t[1][e] = n + e < P.used ? t[1][e] : 0.f;
        }
      }
      activate8<false>(P.act, t[0], c, nullptr);
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] *= t[1][e];
      tile_store8((T*)P.out + at, c);
      if constexpr (kSplits) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float high = to_f32(from_f32<T>(c[e]));
          c[e] = __builtin_isfinite(high) ? c[e] - high : 0.f;
        }
        tile_store8((T*)P.out_low + at, c);
      }
      if (P.kept.gate) {
        Kept8<T>::store(P.kept.gate, at, t[0]);
        Kept8<T>::store(P.kept.up, at, t[1]);
      }
    } else {
      tile_store8((T*)P.out + at, t[0]);
    }
  }
}

// ------------------------------------------------------------------------------------------------- sums of k's shares
struct JoinArgs {
  const float* part[3];
  void* out[3];
  int64_t ldc[3];
  int64_t n[3];              // numbers of a share
  uint32_t row8[3];          // eighths of a row
  int32_t splits;
  Kept kept;                 // kTileGrad
  void* c2;
  int32_t act;
};
template <typename T, int KIND>
__global__ __launch_bounds__(256) void tile_join_kernel(JoinArgs P) {
  constexpr int kMats = KIND == kTileGated ? 2 : 1;
  const int which = blockIdx.y;
  const int64_t n = P.n[which];
  const uint32_t row8 = P.row8[which];
  for (int64_t from = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; from < n; from += (int64_t)gridDim.x * 256 * 8) {
    const uint32_t piece = (uint32_t)(from >> 3), row = piece / row8, col = 8 * (piece - row * row8);   // (the host joins no more than 2^32 pieces)
    float c[kMats][8];
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
      const float* part = P.part[which] + from + (KIND == kTileGated ? ((int64_t)row + m) * (8 * (int64_t)row8) : 0);
      tile_load8(part, c[m]);
#pragma unroll 4
      for (int s = 1; s < P.splits; ++s) {
        float b[8];
        tile_load8(part + s * kMats * n, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) c[m][e] += b[e];
      }
    }
    const int64_t at = row * P.ldc[which] + col;
    if constexpr (KIND == kTileGrad) {
      Kept8<T> gate, up;
      float dg[8], du[8];
      gate.load(P.kept.gate, at);
      up.load(P.kept.up, at);
      gated_grad8(P.act, c[0], gate, up, dg, du);
      tile_store8((T*)P.out[which] + at, dg);
      tile_store8((T*)P.c2 + at, du);
    } else if constexpr (KIND == kTileGated) {
      float h[8];
      activate8<false>(P.act, c[0], h, nullptr);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] *= c[1][e];
      tile_store8((T*)P.out[which] + at, h);
      if (P.kept.gate) {
        Kept8<T>::store(P.kept.gate, at, c[0]);
        Kept8<T>::store(P.kept.up, at, c[1]);
      }
    } else {
      tile_store8((T*)P.out[which] + at, c[0]);
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- copies
// A wave takes a row, or as many neighbouring ones as it has lanes for, by pieces of eight entries: a call with dims that are no multiple of
// eight has one such launch before and one behind its kernels (1503 x 771 and three weights of 771 x 2058 in fp32: 24 MB in and as much out
// in 10.5 us).
struct CopyArgs {
  PalMatrixCopy m[8];
};
template <typename T>
__global__ __launch_bounds__(256) void copy_matrices_kernel(CopyArgs A) {
  const PalMatrixCopy& m = A.m[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, across = (int)min((m.dst_cols + 7) / 8, (int64_t)64), rows = 64 / across;
  const int in_row = lane % across, in_wave = lane / across;
  if (in_wave >= rows) return;
  for (int64_t row = ((int64_t)blockIdx.x * 4 + wave) * rows + in_wave; row < m.dst_rows; row += (int64_t)gridDim.x * 4 * rows) {
    const T* src = (const T*)m.src + row * m.src_ld;
    T* dst = (T*)m.dst + row * m.dst_ld;
    for (int64_t c = 8 * in_row; c < m.dst_cols; c += 8 * across) {
      Piece8<T> b;
      load_piece(b, src + c, row < m.rows ? (int)min(m.cols - c, (int64_t)8) : 0);
      if (c + 8 <= m.dst_cols) {
        b.store(dst + c);
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (c + e < m.dst_cols) dst[c + e] = b.at(e);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- host
// Tiles that the products are made of: 256 x 256 and, for matrices whose columns fill the chip better so, 256 x 192 by eight waves, one
// workgroup a compute unit; 128 x 128 by four, two of them, where there are few tiles; of fp32 rows 64 x 64 (64 x 128 of gated products).
// Products of bf16 rows are bound by the reads and writes of LDS, of which a large tile has less per number; those of fp32 rows by the matrix units,
// whose share of a compute unit a tile of any size uses in full: they take the tiles that spread best, and a unit's tiles count one by one.
// Measured (a kernel between two events, in a pass over the whole block) with 256 x 256, 256 x 192 and 128 x 128: 16384 rows of bf16, 768 -> 2048 gated 127, -,
// 142 us, back to 768 63, 56, 63, gradient of h 112, 131, 117, of x 135, 125, 138, of the weights with shares 185, 200, 206; 8192 rows, 5632 -> 2048 145, 203,
// 197.  1503 rows of fp32, the weights' gradients (771 x 2058, three) with 256, 128 and 64: 193, 148, 146.  Shares of k, with their sum, against none: the
// weights' gradients of the 16384 rows 185 + 13 and 292 us, 48 rows of bf16 2048 -> 5632 gated 17 + 7 and 27, back 14 + 7 and 61.
enum TileForm { kTileBig = 0, kTileNarrow, kTileSmall, kTileTiny, kTileForms };
struct TileShape {
  int m, n, slots;           // of the chip, bf16 rows
  double bf16_us, fp32_us;   // time of a step, measured: while every slot has a tile; of one tile that has a compute unit's matrix units
};
constexpr TileShape kTileShapes[kTileForms] = {{256, 256, 256, 1.65, 7.4}, {256, 192, 256, 1.35, 5.6}, {128, 128, 512, 1.0, 1.95}, {64, 64, 0, 0, 0.52}};
constexpr int tile_cols(int form, int kind) {   // of C
  return kind == kTileGated ? (form == kTileTiny ? 64 : kTileShapes[form].n / 2) : kTileShapes[form].n;
}
struct TilePlan {
  int form, tiles, splits, split_steps;
  double us;
};

// Tile form and shares of k: the cheapest by the time of a step of a tile, the launch's rounds over the chip and, for shares, their way
// through memory.
static TilePlan plan_tiles(const TileArgs& P, int kind, int dtype) {
  TilePlan best{};
  double least = 1e30;
  const int per = dtype == PAL_DTYPE_BF16 ? 64 : 32, one = (P.k + per - 1) / per, steps = kind == kTileTwice ? 2 * one : one;
  double numbers = 0;
  for (int i = 0; i < P.n_prod; ++i) numbers += (double)P.prod[i].a.rows * P.prod[i].b.rows * (kind == kTileGated ? 2 : 1);
  const int most = numbers > 3e10 ? 1 : 32;   // shares (the join counts pieces in 32 bits)
  for (int form = 0; form < kTileForms; ++form) {
    if ((form == kTileNarrow && kind == kTileGated) || (form == kTileTiny && dtype == PAL_DTYPE_BF16)) continue;
    const TileShape& t = kTileShapes[form];
    const int tn = tile_cols(form, kind), slots = dtype == PAL_DTYPE_BF16 ? t.slots : 256;
    int64_t tiles = 0;
    for (int i = 0; i < P.n_prod; ++i)
      tiles += (int64_t)((P.prod[i].a.rows + t.m - 1) / t.m) * ((P.prod[i].b.rows + tn - 1) / tn);
    if (tiles > 1 << 24) continue;
    const double step = dtype == PAL_DTYPE_BF16 ? t.bf16_us : t.fp32_us * (kind == kTileGated && form == kTileTiny ? 2 : 1);
    // (no more shares than fill the chip a few times)
    for (int s = 1; s <= most && s <= steps && (s == 1 || tiles * s <= 8 * (int64_t)slots); ++s) {
      const int share = (steps + s - 1) / s, splits = (steps + share - 1) / share;
      if (splits != s) continue;
      const double rounds = (double)((tiles * s + slots - 1) / slots);
      const double us = rounds * share * step + 3 + (s > 1 ? 4 + numbers * s * (4 / 3.5e6 + 4 / 1e7) : 0);
      if (us < least) {
        least = us;
        best = TilePlan{form, (int)tiles, s, share, us};
      }
    }
  }
  return best;
}

template <typename T, int KIND, bool ACOLS, bool BCOLS, int WM, int WN, int NFM, int NFN>
static int tile_launch(const TileArgs& P, int id, hipStream_t s) {
  constexpr size_t lds = (size_t)2 * 128 * 16 * (NFM * WM + NFN * WN);
  constexpr int slots = 256 * (lds > kMaxLds / 2 ? 1 : lds > kMaxLds / 4 ? 2 : 4);   // workgroups that the chip holds at a time
  const auto kernel = &tile_product_kernel<T, KIND, ACOLS, BCOLS, WM, WN, NFM, NFN>;
  if (int rc = allow_lds((const void*)kernel, lds)) return rc;
  PAL_TIMED_LAUNCH(id, s, (*kernel), dim3(P.tiles * P.splits < slots ? P.tiles * P.splits : slots), dim3(64 * WM * WN), lds, s, P);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

static size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
static size_t part_bytes(const TileArgs& P, const TilePlan& plan, int kind) {
  if (plan.splits < 2) return 0;
  size_t n = 0;
  for (int i = 0; i < P.n_prod; ++i) n += (size_t)P.prod[i].a.rows * P.prod[i].b.rows;
  return round256(n * sizeof(float) * plan.splits * (kind == kTileGated ? 2 : 1));
}

// the launches of one set of products; `part`: part_bytes of them
template <typename T, int KIND, bool ACOLS, bool BCOLS>
static int tile_run(TileArgs P, const TilePlan& plan, float* part, int id, hipStream_t s) {
  if (!plan.tiles) return PAL_E_DIM;
  const int t = kTileShapes[plan.form].m, tn = tile_cols(plan.form, KIND);
  P.tiles = plan.tiles;
  P.splits = plan.splits;
  P.split_steps = plan.split_steps;
  int first = 0;
  JoinArgs J{};
  int64_t most = 0;
  for (int i = 0; i < P.n_prod; ++i) {
    TileProduct& p = P.prod[i];
    p.first = first;
    p.tiles_n = (p.b.rows + tn - 1) / tn;
    first += p.tiles_n * ((p.a.rows + t - 1) / t);
    p.part = part;
    J.part[i] = part;
    J.out[i] = p.c;
    J.ldc[i] = p.ldc;
    J.row8[i] = p.b.rows / 8;
    J.n[i] = (int64_t)p.a.rows * p.b.rows;
    most = J.n[i] > most ? J.n[i] : most;
    if (part) part += J.n[i] * plan.splits * (KIND == kTileGated ? 2 : 1);
  }
  int rc = PAL_OK;
  if (plan.form == kTileBig) rc = tile_launch<T, KIND, ACOLS, BCOLS, 2, 4, 8, 4>(P, id, s);
  else if (plan.form == kTileSmall) rc = tile_launch<T, KIND, ACOLS, BCOLS, 2, 2, 4, 4>(P, id, s);
  else if (plan.form == kTileTiny) {
    if constexpr (sizeof(T) == 4) rc = tile_launch<T, KIND, ACOLS, BCOLS, 2, 2, 2, KIND == kTileGated ? 4 : 2>(P, id, s);
  } else if constexpr (KIND != kTileGated) {
    rc = tile_launch<T, KIND, ACOLS, BCOLS, 4, 2, 4, 6>(P, id, s);
  }
  if (rc || plan.splits < 2) return rc;
  J.splits = plan.splits; J.kept = P.kept; J.c2 = P.c2; J.act = P.act;
  const int64_t blocks = (most + 2047) / 2048;
  PAL_TIMED_LAUNCH(kKernTileJoin, s, (tile_join_kernel<T, KIND>), dim3((unsigned)(blocks < 4096 ? blocks : 4096), P.n_prod),
                   dim3(256), 0, s, J);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

template <typename T, bool GATED, int R>
static int few_launch_rows(const FewArgs& P, hipStream_t s) {
  constexpr int kMost = GATED ? 8 : 16, kGo = R == 1 ? kFewSpans : kFewSpans / 2;
  const int spans = (P.k + 8 * TileType<T>::kPiece - 1) / (8 * TileType<T>::kPiece);
  const int rounds = (spans + kGo * kMost - 1) / (kGo * kMost), waves = (spans + kGo * rounds - 1) / (kGo * rounds);
  const dim3 grid((P.n + 15) / 16), block(64 * waves);
  const size_t lds = (size_t)waves * (GATED ? 2 : 1) * R * 64 * sizeof(f32x4);
  const int id = GATED ? kKernMlpFewUp : kKernMlpFewDown;
  PAL_TIMED_LAUNCH(id, s, (few_rows_kernel<T, GATED, R>), grid, block, lds, s, P);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
template <typename T, bool GATED>
static int few_launch(const FewArgs& P, hipStream_t s) {
  const int groups = (P.rows + 15) / 16;
  return groups == 1   ? few_launch_rows<T, GATED, 1>(P, s)
         : groups == 2 ? few_launch_rows<T, GATED, 2>(P, s)
         : groups == 3 ? few_launch_rows<T, GATED, 3>(P, s)
                       : few_launch_rows<T, GATED, 4>(P, s);
}

static int check_mlp(const PalMlpDims* d) {
  if (!d) return PAL_E_NULL;
  if (d->dtype != PAL_DTYPE_F32 && d->dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->activation < 0 || d->activation > PAL_ACT_RELU) return PAL_E_DIM;
  for (int32_t n : {d->dim, d->hidden, d->out_dim})
    if (n <= 0 || n % 8 || n > 1 << 20) return PAL_E_DIM;
  if (d->hidden_pad < 0 || d->hidden_pad > 7) return PAL_E_DIM;
  if (d->rows <= 0 || d->rows > 1 << 30 || d->x_stride < d->dim || d->x_stride % 8) return PAL_E_DIM;
  // a tile's rows are reached by offsets of 31 bits from its first
  if (d->x_stride > (int64_t)1 << 20) return PAL_E_DIM;
  return PAL_OK;
}
static size_t mlp_elem(const PalMlpDims* d) { return d->dtype == PAL_DTYPE_BF16 ? 2 : 4; }

static TileOperand operand(const void* p, int64_t ld_elems, size_t es, int64_t rows, const void* p2 = nullptr) {
  return TileOperand{(const char*)p, (const char*)p2, (int64_t)(ld_elems * es), (int32_t)rows};
}

// Rows of hidden numbers that the calls lay out themselves (h, dg, du, the kept factors) are an odd number of 128-byte lines apart: rows at a
// multiple of 4096 bytes are in few of the caches' channels, and a tile reads or writes one piece of each of its rows at a time.
static int64_t hidden_ld(const PalMlpDims* d) {
  const int64_t line = 128 / (int64_t)mlp_elem(d), lines = (d->hidden + line - 1) / line;
  return d->hidden < 8 * line ? d->hidden : (lines | 1) * line;
}
static size_t rows_bytes(const PalMlpDims* d) { return round256((size_t)d->rows * hidden_ld(d) * mlp_elem(d)); }
// what the forward call keeps for the backward: the factors, and h
static Kept kept_in(const PalMlpDims* d, void* kept) { return kept ? Kept{kept, (char*)kept + rows_bytes(d)} : Kept{}; }
static void* kept_h(const PalMlpDims* d, void* kept) { return (char*)kept + 2 * rows_bytes(d); }

struct MlpPlan {
  TileArgs up{}, down{}, grad{}, dx{}, dw{};
  TilePlan p_up{}, p_down{}, p_grad{}, p_dx{}, p_dw{};
};
static void plan_fwd(const PalMlpDims* d, const PalMlpTensors* t, const void* h, MlpPlan& m) {
  const size_t es = mlp_elem(d);
  const int64_t ld = hidden_ld(d);
  m.up.n_prod = 1;
  m.up.k = d->dim;
  m.up.prod[0].a = operand(t->x, d->x_stride, es, d->rows);
  m.up.prod[0].b = operand(t->w_gate, d->dim, es, d->hidden, t->w_up);
  m.up.prod[0].c = (void*)h;
  m.up.prod[0].ldc = ld;
  m.up.kept = kept_in(d, t->kept);
  m.up.act = d->activation;
  m.up.used = d->hidden - d->hidden_pad;
  m.down.n_prod = 1;
  m.down.k = d->hidden;
  m.down.prod[0].a = operand(h, ld, es, d->rows);
  m.down.prod[0].b = operand(t->w_down, d->hidden, es, d->out_dim);
  m.down.prod[0].c = t->y;
  m.down.prod[0].ldc = d->out_dim;
  m.p_up = plan_tiles(m.up, kTileGated, d->dtype);
  m.p_down = plan_tiles(m.down, kTilePlain, d->dtype);
}
// the gradient of h, and dg and du with it, is for these; that of w_down takes h alone
static bool wants_dh(const PalMlpGrads* g) { return g->dx || g->dw_gate || g->dw_up; }
static void plan_bwd(const PalMlpDims* d, const PalMlpTensors* t, const PalMlpGrads* g, void* dg, void* du, MlpPlan& m) {
  const size_t es = mlp_elem(d);
  const int64_t ld = hidden_ld(d);
  m.grad.n_prod = 1;
  m.grad.k = d->out_dim;
  m.grad.prod[0].a = operand(g->dy, d->out_dim, es, d->rows);
  m.grad.prod[0].b = operand(t->w_down, d->hidden, es, d->hidden);
  m.grad.prod[0].c = dg;
  m.grad.prod[0].ldc = ld;
  m.grad.kept = kept_in(d, t->kept);
  m.grad.c2 = du;
  m.grad.act = d->activation;
  m.grad.used = d->hidden - d->hidden_pad;
  if (wants_dh(g)) m.p_grad = plan_tiles(m.grad, kTileGrad, d->dtype);
  m.dx.n_prod = 1;
  m.dx.k = d->hidden;
  m.dx.prod[0].a = operand(dg, ld, es, d->rows, du);
  m.dx.prod[0].b = operand(t->w_gate, d->dim, es, d->dim, t->w_up);
  m.dx.prod[0].c = g->dx;
  m.dx.prod[0].ldc = d->dim;
  if (g->dx) m.p_dx = plan_tiles(m.dx, kTileTwice, d->dtype);
  m.dw.k = (int32_t)d->rows;
  auto add = [&](const TileOperand& a, const TileOperand& b, void* c) {
    if (!c) return;
    TileProduct& p = m.dw.prod[m.dw.n_prod++];
    p.a = a;
    p.b = b;
    p.c = c;
    p.ldc = b.rows;
  };
  add(operand(dg, ld, es, d->hidden), operand(t->x, d->x_stride, es, d->dim), g->dw_gate);
  add(operand(du, ld, es, d->hidden), operand(t->x, d->x_stride, es, d->dim), g->dw_up);
  add(operand(g->dy, d->out_dim, es, d->out_dim), operand(kept_h(d, t->kept), ld, es, d->hidden), g->dw_down);
  if (m.dw.n_prod) m.p_dw = plan_tiles(m.dw, kTilePlain, d->dtype);
}
static size_t most_of(size_t a, size_t b) { return a > b ? a : b; }

// Plans a forward call; true: it takes the kernel of few rows.  Beyond 16 rows that goes by its time, fitted to 17 to 64 rows of six sizes (256 -> 704 -> 256 to 2048 -> 5632 -> 2048; within
// a sixth), against that of the tiles' plan, which is up to a quarter too low there.  bf16, 33 rows: 768 -> 2048 -> 768 14.0 us and 22.4 by tiles, 1536 -> 4096 23.7 and 31.6, 2048 -> 5632 38.1 and
// 32.5; fp32, 32 rows: 512 -> 1408 16.9 and 22.1, 1024 -> 2816 30.5 and 29.5.
static bool plan_few(const PalMlpDims* d, const PalMlpTensors* t, const void* h, MlpPlan& m) {
  if (d->rows <= 16) return true;
  plan_fwd(d, t, h, m);
  if (d->rows > kFewRows) return false;
  auto rounds = [](int n) { return (double)((n + 16 * 256 - 1) / (16 * 256)); };   // of workgroups of sixteen columns over the compute units
  const double k_bytes = (rounds(d->hidden) * d->dim + rounds(d->out_dim) * d->hidden) * (double)mlp_elem(d);
  return 5 + k_bytes * (0.00086 + 0.00003 * (double)d->rows) < 1.25 * (m.p_up.us + m.p_down.us);
}

template <typename T>
static int mlp_fwd(const PalMlpDims* d, const PalMlpTensors* t, char* ws, hipStream_t s) {
  void* h = t->kept ? kept_h(d, t->kept) : ws;
  MlpPlan m;
  if (plan_few(d, t, h, m)) {
    const int64_t ld = hidden_ld(d);
    void* low = t->kept ? ws : ws + rows_bytes(d);
    FewArgs up{t->x, t->w_gate, t->w_up, h, kept_in(d, t->kept), d->x_stride, ld, (int32_t)d->rows, d->hidden, d->dim, d->activation, nullptr, low,
               d->hidden - d->hidden_pad};
    if (int rc = few_launch<T, true>(up, s)) return rc;
    FewArgs down{h, t->w_down, nullptr, t->y, Kept{}, ld, d->out_dim, (int32_t)d->rows, d->out_dim, d->hidden, 0, low, nullptr, 0};
    return few_launch<T, false>(down, s);
  }
  float* part = (float*)(t->kept ? ws : ws + rows_bytes(d));
  if (int rc = tile_run<T, kTileGated, false, false>(m.up, m.p_up, part, kKernMlpUp, s)) return rc;
  return tile_run<T, kTilePlain, false, false>(m.down, m.p_down, part, kKernMlpDown, s);
}
template <typename T>
static int mlp_bwd(const PalMlpDims* d, const PalMlpTensors* t, const PalMlpGrads* g, char* ws, hipStream_t s) {
  const size_t n = wants_dh(g) ? rows_bytes(d) : 0;
  MlpPlan m;
  plan_bwd(d, t, g, ws, ws + n, m);
  float* part = (float*)(ws + 2 * n);
  if (wants_dh(g))
    if (int rc = tile_run<T, kTileGrad, false, true>(m.grad, m.p_grad, part, kKernMlpGrad, s)) return rc;
  if (g->dx)
    if (int rc = tile_run<T, kTileTwice, false, true>(m.dx, m.p_dx, part, kKernMlpDx, s)) return rc;
  if (m.dw.n_prod) return tile_run<T, kTilePlain, true, true>(m.dw, m.p_dw, part, kKernMlpDw, s);
  return PAL_OK;
}

}  // namespace pal

extern "C" int pal_copy_matrices(const PalMatrixCopy* m, int32_t n, int32_t dtype, void* stream) {
  using namespace pal;
  if (!m) return PAL_E_NULL;
  if (dtype != PAL_DTYPE_F32 && dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (n < 1 || n > 8) return PAL_E_DIM;
  CopyArgs A{};
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    A.m[i] = m[i];
    if (!m[i].src || !m[i].dst) return PAL_E_NULL;
    if (m[i].rows < 1 || m[i].cols < 1 || m[i].rows > m[i].dst_rows || m[i].cols > m[i].dst_cols || m[i].dst_rows > 1 << 30 || m[i].dst_cols > 1 << 30 ||
        m[i].src_ld < m[i].cols || m[i].dst_ld < m[i].dst_cols)
      return PAL_E_DIM;
    const int64_t across = (m[i].dst_cols + 7) / 8 < 64 ? (m[i].dst_cols + 7) / 8 : 64, per = 4 * (64 / across), blocks = (m[i].dst_rows + per - 1) / per;
    most = blocks > most ? blocks : most;
  }
  const dim3 grid((unsigned)(most < 2048 ? most : 2048), n);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PAL_DTYPE_BF16) PAL_TIMED_LAUNCH(kKernCopyMatrices, s, copy_matrices_kernel<bf16_t>, grid, dim3(256), 0, s, A);
  else PAL_TIMED_LAUNCH(kKernCopyMatrices, s, copy_matrices_kernel<float>, grid, dim3(256), 0, s, A);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

extern "C" int pal_gated_mlp_forms(const PalMlpDims* d, const PalMlpGrads* g, PalMlpForms* forms) {
  using namespace pal;
  if (int rc = check_mlp(d)) return rc;
  if (!forms) return PAL_E_NULL;
  *forms = PalMlpForms{};
  MlpPlan m;
  PalMlpTensors t{};
  auto put = [&](int i, const TilePlan& p, int kind) {
    if (!p.tiles) return;
    forms->tile_rows[i] = kTileShapes[p.form].m;
    forms->tile_cols[i] = tile_cols(p.form, kind);
    forms->shares[i] = p.splits;
    forms->tiles[i] = p.tiles;
  };
  if (!plan_few(d, &t, nullptr, m)) {
    put(0, m.p_up, kTileGated);
    put(1, m.p_down, kTilePlain);
  }
  if (!g) return PAL_OK;
  plan_bwd(d, &t, g, nullptr, nullptr, m);
  put(2, m.p_grad, kTileGrad);
  put(3, m.p_dx, kTileTwice);
  put(4, m.p_dw, kTilePlain);
  return PAL_OK;
}
extern "C" size_t pal_gated_mlp_kept_bytes(const PalMlpDims* d) {
  using namespace pal;
  return check_mlp(d) == PAL_OK ? 3 * rows_bytes(d) : 0;
}
extern "C" size_t pal_gated_mlp_fwd_workspace_bytes(const PalMlpDims* d, int keeps) {
  using namespace pal;
  if (check_mlp(d) != PAL_OK) return 0;
  const size_t h = keeps ? 0 : rows_bytes(d);
  MlpPlan m;
  PalMlpTensors t{};
  if (plan_few(d, &t, nullptr, m)) return h + (d->dtype == PAL_DTYPE_BF16 && d->rows <= 16 ? rows_bytes(d) : 0);
  return h + most_of(part_bytes(m.up, m.p_up, kTileGated), part_bytes(m.down, m.p_down, kTilePlain));
}
extern "C" int pal_gated_mlp_fwd(const PalMlpDims* d, const PalMlpTensors* t, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pal;
  if (int rc = check_mlp(d)) return rc;
  if (!t || !t->x || !t->w_gate || !t->w_up || !t->w_down || !t->y) return PAL_E_NULL;
  for (const void* p : {t->x, t->w_gate, t->w_up, t->w_down, (const void*)t->y, (const void*)t->kept})
    if (!is_aligned16(p)) return PAL_E_ALIGN;
  const size_t need = pal_gated_mlp_fwd_workspace_bytes(d, t->kept != nullptr);
  if (need && (!workspace || workspace_bytes < need)) return PAL_E_WORKSPACE;
  if (!is_aligned16(workspace)) return PAL_E_ALIGN;
  return d->dtype == PAL_DTYPE_BF16 ? mlp_fwd<bf16_t>(d, t, (char*)workspace, (hipStream_t)stream)
                                    : mlp_fwd<float>(d, t, (char*)workspace, (hipStream_t)stream);
}
extern "C" size_t pal_gated_mlp_bwd_workspace_bytes(const PalMlpDims* d, const PalMlpGrads* g) {
  using namespace pal;
  if (check_mlp(d) != PAL_OK || !g) return 0;
  MlpPlan m;
  PalMlpTensors t{};
  plan_bwd(d, &t, g, nullptr, nullptr, m);
  const size_t part = most_of(part_bytes(m.dx, m.p_dx, kTileTwice), part_bytes(m.dw, m.p_dw, kTilePlain));
  return (wants_dh(g) ? 2 * rows_bytes(d) : 0) + most_of(part_bytes(m.grad, m.p_grad, kTileGrad), part);
}
extern "C" int pal_gated_mlp_bwd(const PalMlpDims* d, const PalMlpTensors* t, const PalMlpGrads* g, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  using namespace pal;
  if (int rc = check_mlp(d)) return rc;
  if (!t || !t->x || !t->w_gate || !t->w_up || !t->w_down || !t->kept || !g || !g->dy) return PAL_E_NULL;
  for (const void* p : {t->x, t->w_gate, t->w_up, t->w_down, (const void*)t->kept, g->dy, (const void*)g->dx, (const void*)g->dw_gate,
                        (const void*)g->dw_up, (const void*)g->dw_down})
    if (!is_aligned16(p)) return PAL_E_ALIGN;
  const size_t need = pal_gated_mlp_bwd_workspace_bytes(d, g);
  if (need && (!workspace || workspace_bytes < need)) return PAL_E_WORKSPACE;
  if (!is_aligned16(workspace)) return PAL_E_ALIGN;
  return d->dtype == PAL_DTYPE_BF16 ? mlp_bwd<bf16_t>(d, t, g, (char*)workspace, (hipStream_t)stream)
                                    : mlp_bwd<float>(d, t, g, (char*)workspace, (hipStream_t)stream);
}
