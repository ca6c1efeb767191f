// Layer norm, alone or as a pre-norm with a dropout and the residual's addition in front of it:
//     s = dropout(x) + residual (rounded to the residual stream's type, handed on),   h = (s - mean s) r,   y = h w + b,
//     r = 1 / sqrt(mean (s - mean s)^2 + eps).
// Backward, with dy and the gradient dres that comes back along the stream (both may be missing):
//     ds = r (w dy - mean(w dy) - h mean(w dy h)) + dres  (the gradient of residual; dropped and scaled as x was, that of x),
//     dw = sum over rows of dy h,   db = sum over rows of dy.
// It reads s as the forward call handed it on (or x, where s is x), and the row's mean and r, which the forward call keeps.
//
// Bound by HBM: every row is read once and written once, as in residual_norm.hip, whose division of the work this has: one wave holds a
// row of up to 2048 entries, four one of up to 16384, the next row is fetched before the present one is summed.  The variance is
// that of the row in registers around its mean, in a second sum: no difference of large squares.  Dropout's words are made from the place
// (philox.h); pieces of rows whose length is no multiple of eight are then not moved back, so that four words belong to one piece.  16384 rows of
// 1536, bf16 with a dropout beside an fp32 stream: forward 302 MB in 61 us, backward 403 MB in 77, its sum over the workgroups' shares 5.
#include "norm_rows.h"
#include "pal_common.h"
#include "pal_host.h"
#include "pal_profile.h"
#include "philox.h"

namespace pal {

struct LayerNormArgs {
  const void *x, *res, *weight, *bias;
  void *s, *y;            // s: NULL where it is x itself
  float* stats;           // [rows][2] or NULL
  const void *dy, *dres;
  void *dx, *ds;          // ds: NULL (not wanted, or dx)
  float *part, *dweight, *dbias;  // part: [workgroups][2][dim]
  int64_t rows, x_stride, res_stride;
  int dim, weight_bf16;
  float eps;
  DropArgs drop;
};

// A row's beginning in scalar registers, and a lane's place in it by 32 bits, which a load or store adds itself.  (As pointers of the lanes, 64 bits for
// each piece of each tensor, they were the registers that the backward kernel lacked: read back from scratch memory between the loads of the next
// row, they made each of these wait for the one before.)
template <typename T>
__device__ __forceinline__ T* row_at(T* p, int64_t entries) {
  auto row = (__attribute__((address_space(1))) T*)(p + entries);
  asm("" : "+s"(row));
  return (T*)row;
}
template <typename T>
__device__ __forceinline__ T* lane_at(T* row, int at) { return (T*)((char*)row + (uint32_t)at * (uint32_t)sizeof(T)); }
template <typename T>
__device__ __forceinline__ const T* lane_at(const T* row, int at) { return (const T*)((const char*)row + (uint32_t)at * (uint32_t)sizeof(T)); }
template <bool WHOLE, typename T>
__device__ __forceinline__ void fetch_piece(Piece8<T>& d, const T* row, int at, int D) {
  if constexpr (WHOLE) d.load(lane_at(row, at));
  else load_piece(d, lane_at(row, at), D - at);
}

// entry e of a piece is the row's own and counted here
template <typename At, bool WHOLE>
__device__ __forceinline__ bool counts(const At& p, int e, int D) { return WHOLE ? e >= p.from : p.at + e < D; }

template <typename TX, typename TR, int NV, int WPR, bool DROP, bool WHOLE>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(LayerNormArgs A) {
  typedef NormPiece<NV, WPR, WHOLE> At;
  __shared__ float sMean[2][4], sVar[2][4];
  constexpr int kSlots = 4 / WPR, kStep = 64 * WPR;
  constexpr bool kAll = !WHOLE;                        // every piece may be cut short
  const int slot = WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
  const int lane = threadIdx.x & (kStep - 1);
  const int D = A.dim;
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kSlots;
  int64_t row = (int64_t)blockIdx.x * kSlots + slot;
  if (WPR == 1 && row >= A.rows) return;
  const DropKey key(A.drop);
  float w[NV][8], b[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const At p(lane, v, D);
#pragma unroll
    for (int e = 0; e < 8; ++e) b[v][e] = 0.f;
    if constexpr (WHOLE) {
      load_params(w[v], A.weight, p.at, A.weight_bf16);
      if (A.bias) load_params(b[v], A.bias, p.at, A.weight_bf16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[v][e] = p.at + e < D ? load_rt(A.weight, p.at + e, A.weight_bf16) : 0.f;
        if (A.bias) b[v][e] = p.at + e < D ? load_rt(A.bias, p.at + e, A.weight_bf16) : 0.f;
      }
    }
  }
  Piece8<TX> xb[NV];
  Piece8<TR> rb[NV];
  const bool has_res = A.res != nullptr;
  auto fetch = [&](int64_t r) {
    const TX* x_row = row_at((const TX*)A.x, r * A.x_stride);
    const TR* res_row = row_at((const TR*)A.res, has_res ? r * A.res_stride : 0);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      fetch_piece<WHOLE>(xb[v], x_row, p.at, D);
      if (has_res) fetch_piece<WHOLE>(rb[v], res_row, p.at, D);
    }
  };
  fetch(row);
  for (int turn = 0; row < A.rows; row += step, turn ^= 1) {
    float s[NV][8], sum = 0.f;
    TR* s_row = row_at((TR*)A.s, A.s ? row * D : 0);
    TX* y_row = row_at((TX*)A.y, row * D);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[v][e] = xb[v].get(e);
      if constexpr (DROP) drop_piece(s[v], lane + kStep * v, row, A.drop, key);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (has_res) s[v][e] += rb[v].get(e);
      if (A.s && p.on) store_piece(lane_at(s_row, p.at), s[v], WHOLE ? 8 : D - p.at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[v][e] = to_f32(from_f32<TR>(s[v][e]));   // the norm is that of the stream as it is handed on
        const float q = sum + s[v][e];
        sum = (kAll || At::masked(v)) && !counts<At, WHOLE>(p, e, D) ? sum : q;
      }
    }
    if (row + step < A.rows) fetch(row + step);
    const float mean = row_sum<WPR>(sum, sMean, turn) * inv_d;
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[v][e] -= mean;
        const float q = fmaf(s[v][e], s[v][e], ss);
        ss = (kAll || At::masked(v)) && !counts<At, WHOLE>(p, e, D) ? ss : q;
      }
    }
    ss = row_sum<WPR>(ss, sVar, turn);
    const float r = rsqrtf(fmaf(ss, inv_d, A.eps));
    if (A.stats && lane == 0) {
      f32x2 st = {mean, r};
      *(f32x2*)(A.stats + 2 * row) = st;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fmaf(s[v][e] * r, w[v][e], b[v][e]);
      if (p.on) store_piece(lane_at(y_row, p.at), y, WHOLE ? 8 : D - p.at);
    }
  }
}

template <typename TX, typename TR, int NV, int WPR, bool DROP, bool WHOLE>
__global__ __launch_bounds__(256, WPR == 1 && NV <= 3 ? 2 : 1) void layer_norm_bwd_kernel(LayerNormArgs A) {
  typedef NormPiece<NV, WPR, WHOLE> At;
  __shared__ float sSum[2][4], sDot[2][4];
  extern __shared__ float sW[];   // WPR == 1: [4 waves][512 NV] shares of dweight, then of dbias
  constexpr int kSlots = 4 / WPR, kStep = 64 * WPR;
  constexpr bool kAll = !WHOLE;
  const int slot = WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
  const int lane = threadIdx.x & (kStep - 1);
  const int D = A.dim;
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kSlots;
  const bool has_dy = A.dy != nullptr, has_dres = A.dres != nullptr;
  const int64_t s_stride = A.s ? D : A.x_stride;
  const TR* s_rows = A.s ? (const TR*)A.s : (const TR*)A.x;
  const DropKey key(A.drop);
  constexpr bool kWide = NV == 8;   // rows whose weights and whose next one would not fit the registers as well: both are read when they are used
  float w[kWide ? 1 : NV][8], dw[NV][8], db[NV][8];
  auto weights = [&](int v) {
    const At p(lane, v, D);
    float (&o)[8] = w[kWide ? 0 : v];
    if constexpr (WHOLE) {
      load_params(o, A.weight, p.at, A.weight_bf16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = p.at + e < D ? load_rt(A.weight, p.at + e, A.weight_bf16) : 0.f;
    }
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (!kWide) weights(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[v][e] = db[v][e] = 0.f;
  }
  Piece8<TR> sb[NV], eb[NV];
  Piece8<TX> gb[NV];
  f32x2 st;
  auto fetch = [&](int64_t r) {
    st = *(const f32x2*)(A.stats + 2 * r);
    const TR* s_row = row_at(s_rows, r * s_stride);
    const TX* dy_row = row_at((const TX*)A.dy, has_dy ? r * D : 0);
    const TR* dres_row = row_at((const TR*)A.dres, has_dres ? r * D : 0);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      fetch_piece<WHOLE>(sb[v], s_row, p.at, D);
      if (has_dy) fetch_piece<WHOLE>(gb[v], dy_row, p.at, D);
      if (has_dres) fetch_piece<WHOLE>(eb[v], dres_row, p.at, D);
    }
  };
  int64_t row = (int64_t)blockIdx.x * kSlots + slot;
  if (!kWide && row < A.rows) fetch(row);
  for (int turn = 0; row < A.rows; row += step, turn ^= 1) {
    if constexpr (kWide) fetch(row);
    float h[NV][8], sum = 0.f, dot = 0.f;
    const float mean = st[0], r = st[1];
    Piece8<TX> gk[NV];       // (as they were read: half the registers of bf16 rows)
    Piece8<TR> ek[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      const float (&wv)[8] = w[kWide ? 0 : v];
      if (kWide) weights(v);
      gk[v] = gb[v];
      ek[v] = eb[v];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[v][e] = (sb[v].get(e) - mean) * r;
        const float gw = (has_dy ? gk[v].get(e) : 0.f) * wv[e], q = sum + gw, d = fmaf(gw, h[v][e], dot);
        const bool out = (kAll || At::masked(v)) && !counts<At, WHOLE>(p, e, D);
        sum = out ? sum : q;
        dot = out ? dot : d;
      }
    }
    if (!kWide && row + step < A.rows) fetch(row + step);
    sum = row_sum<WPR>(sum, sSum, turn) * inv_d;
    dot = row_sum<WPR>(dot, sDot, turn) * inv_d;
    TR* ds_row = row_at((TR*)A.ds, A.ds ? row * D : 0);
    TX* dx_row = row_at((TX*)A.dx, row * D);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      float d[8];
      const float (&wv)[8] = w[kWide ? 0 : v];
      if (kWide) weights(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = has_dy ? gk[v].get(e) : 0.f, ex = has_dres ? ek[v].get(e) : 0.f;
        dw[v][e] = fmaf(g, h[v][e], dw[v][e]);
        db[v][e] += g;
        d[e] = has_dy ? fmaf(r, fmaf(-h[v][e], dot, fmaf(g, wv[e], -sum)), ex) : ex;
      }
      if (p.on && A.ds) store_piece(lane_at(ds_row, p.at), d, WHOLE ? 8 : D - p.at);
      if constexpr (DROP) drop_piece(d, lane + kStep * v, row, A.drop, key);
      if (p.on) store_piece(lane_at(dx_row, p.at), d, WHOLE ? 8 : D - p.at);
      if constexpr (DROP || kWide) __builtin_amdgcn_sched_barrier(0);   // (one piece's words and weights at a time)
    }
  }
  // the parameters' gradients: the waves' shares in their order
  float* part = A.part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if constexpr (WPR == 1) {
      if (which) __syncthreads();
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const At p(lane, v, D);
        if (p.on) store_piece(sW + slot * NV * 512 + p.at, which ? db[v] : dw[v], WHOLE ? 8 : D - p.at);
      }
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += 256) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) t += sW[k * NV * 512 + c];
        part[which * D + c] = t;
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const At p(lane, v, D);
        if (p.on) store_piece(part + which * D + p.at, which ? db[v] : dw[v], WHOLE ? 8 : D - p.at);
      }
    }
  }
}

// dweight and dbias: 64 groups of sixteen threads take sixteen columns, each group its share of the workgroups in order.  In 64 bits: the sums of
// up to 1024 shares would cost most of the bits that the waves' sums of a few rows leave (4099 rows of 1531 in fp32, errors of the norm: 1.2e-7 and 1.1e-7 in 32 bits, 7.6e-8 and 5.8e-8 so; no slower).
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* part, float* dweight, float* dbias, int n, int dim) {
  __shared__ double s[64][17];
  const int x = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + x, all = 2 * dim;
  double t = 0.0;
  if (c < all) {
#pragma unroll 8
    for (int j = g; j < n; j += 64) t += part[(int64_t)j * all + c];
  }
  s[g][x] = t;
  __syncthreads();
  if (g < 8) {
    t = s[8 * g][x];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += s[8 * g + k][x];
  }
  __syncthreads();
  if (g < 8) s[g][x] = t;
  __syncthreads();
  if (g == 0 && c < all) {
    t = s[0][x];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += s[k][x];
    if (c < dim) dweight[c] = (float)t;
    else if (dbias) dbias[c - dim] = (float)t;
  }
}

static int layer_norm_blocks(int64_t rows, int dim, bool bwd) {
  const int slots = dim > 2048 ? 1 : 4;
  // Backward: as many as the chip holds at a time, by the registers that a row's pieces take: every further one is a share more of the parameters'
  // gradients, and with fewer a compute unit waits (16384 rows of bf16, between two events: of 2048, 40 us with 256 and 46 with 512; of 1536 beside an
  // fp32 stream, with a dropout, 83 and 81).
  const bool two = dim <= 1536 || (dim > 2048 && dim <= 4096);
  const int64_t want = (rows + slots - 1) / slots, most = !bwd ? 2048 : dim <= 512 ? 1024 : two ? 512 : 256;
  return (int)(want < most ? want : most);
}

template <typename TX, typename TR, bool BWD, bool DROP>
static void layer_norm_launch(const LayerNormArgs& A, hipStream_t s) {
  const dim3 grid(layer_norm_blocks(A.rows, A.dim, BWD));
  const bool wide = A.dim > 2048;
  const int nv = (A.dim + (wide ? 2047 : 511)) / (wide ? 2048 : 512);
#define PAL_NORM(NV, WPR, WHOLE)                                                                                      \
  do {                                                                                                             \
    if constexpr (BWD) {                                                                                           \
      const size_t lds = WPR == 1 ? (size_t)4 * 512 * NV * sizeof(float) : 0;                                      \
      PAL_TIMED_LAUNCH(kKernLayerNormBwd, s, (layer_norm_bwd_kernel<TX, TR, NV, WPR, DROP, WHOLE>), grid, dim3(256), lds, s, A); \
    } else {                                                                                                       \
      PAL_TIMED_LAUNCH(kKernLayerNormFwd, s, (layer_norm_fwd_kernel<TX, TR, NV, WPR, DROP, WHOLE>), grid, dim3(256), 0, s, A); \
    }                                                                                                              \
  } while (0)
#define PAL_NORM_ROWS(WHOLE)                                                                                          \
  do {                                                                                                             \
    if (!wide) {                                                                                                   \
      if (nv == 1) PAL_NORM(1, 1, WHOLE);                                                                            \
      else if (nv == 2) PAL_NORM(2, 1, WHOLE);                                                                       \
      else if (nv == 3) PAL_NORM(3, 1, WHOLE);                                                                       \
      else PAL_NORM(4, 1, WHOLE);                                                                                    \
    } else {                                                                                                       \
      if (nv <= 2) PAL_NORM(2, 4, WHOLE);                                                                            \
      else if (nv <= 4) PAL_NORM(4, 4, WHOLE);                                                                       \
      else PAL_NORM(8, 4, WHOLE);                                                                                    \
    }                                                                                                              \
  } while (0)
  if constexpr (DROP) {
    if (A.dim % 8 == 0) PAL_NORM_ROWS(true);
    else PAL_NORM_ROWS(false);
  } else {
    if (A.dim < 8) PAL_NORM(1, 1, false);
    else PAL_NORM_ROWS(true);
  }
#undef PAL_NORM_ROWS
#undef PAL_NORM
}
template <bool BWD>
static void layer_norm_dispatch(const PalLayerNormDims* d, const LayerNormArgs& A, hipStream_t s) {
  const bool drop = d->drop.p > 0.0;
  if (d->dtype == PAL_DTYPE_F32) drop ? layer_norm_launch<float, float, BWD, true>(A, s) : layer_norm_launch<float, float, BWD, false>(A, s);
  else if (d->res_dtype == PAL_DTYPE_F32) drop ? layer_norm_launch<bf16_t, float, BWD, true>(A, s) : layer_norm_launch<bf16_t, float, BWD, false>(A, s);
  else drop ? layer_norm_launch<bf16_t, bf16_t, BWD, true>(A, s) : layer_norm_launch<bf16_t, bf16_t, BWD, false>(A, s);
}

static int layer_norm_args(const PalLayerNormDims* d, LayerNormArgs& A) {
  if (!d) return PAL_E_NULL;
  if (d->rows <= 0 || d->dim <= 0 || d->dim > kNormMaxRow || d->rows > (int64_t)1 << 40) return PAL_E_DIM;
  if (d->dtype != PAL_DTYPE_F32 && d->dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->res_dtype != PAL_DTYPE_F32 && d->res_dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->dtype == PAL_DTYPE_F32 && d->res_dtype != PAL_DTYPE_F32) return PAL_E_DTYPE;
  if (d->weight_dtype != PAL_DTYPE_F32 && d->weight_dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->x_stride < d->dim || d->res_stride < d->dim) return PAL_E_DIM;
  if (!(d->eps >= 0.f)) return PAL_E_DIM;
  A.rows = d->rows; A.dim = d->dim; A.weight_bf16 = d->weight_dtype == PAL_DTYPE_BF16; A.eps = d->eps;
  A.x_stride = d->x_stride; A.res_stride = d->res_stride;
  return drop_args(d->drop, A.drop);
}

// ------------------------------------------------------------------------------------------------------------- dropout
struct DropoutArgs {
  const void* x;
  void* y;
  int64_t pieces, stride;     // of all rows; elements between rows of x
  uint32_t dim, per_row, magic;
  int turns;
  DropArgs drop;
};

// A workgroup takes `turns` times 256 neighbouring pieces of eight entries; pieces are numbered over the rows.  Bound by HBM: 16384 rows of 2048 in
// bf16 are 134 MB in 25.8 us (5.2 TB/s), the vector units at work for a half of it, most of that on the random words.  Two turns once they fill the
// chip: 25.8 us, where one is 27.2, four 27.1 and sixteen 30.9.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs A) {
  const DropKey key(A.drop);
  const int64_t first = (int64_t)blockIdx.x * 256 * A.turns;
  // the workgroup's first row and its place in it; from there on 32 bits are enough
  int64_t row0;
  uint32_t in_row;
  if (A.pieces < (int64_t)1 << 31) {
    row0 = (uint32_t)first / A.per_row;
    in_row = (uint32_t)first - (uint32_t)row0 * A.per_row;
  } else {
    row0 = first / A.per_row;
    in_row = (uint32_t)(first - row0 * A.per_row);
  }
  for (int t = 0; t < A.turns; ++t) {
    const uint32_t i = t * 256 + threadIdx.x;
    if (first + i >= A.pieces) return;
    // (in_row + i) / per_row: the product by 2^32 / per_row, rounded up, is at most one too high
    const uint32_t n = in_row + i;
    uint32_t q = A.per_row > 1 ? __umulhi(n, A.magic) : n;
    if (q * (uint64_t)A.per_row > n) --q;
    const uint32_t piece = n - q * A.per_row;
    const int64_t row = row0 + q;
    const int left = (int)(A.dim - 8 * piece);
    Piece8<T> b;
    load_piece(b, (const T*)A.x + row * A.stride + 8 * (int64_t)piece, left);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = b.get(e);
    drop_piece(x, piece, row, A.drop, key);
    store_piece((T*)A.y + row * (int64_t)A.dim + 8 * (int64_t)piece, x, left);
  }
}

}  // namespace pal

extern "C" int pal_layer_norm_fwd(const PalLayerNormDims* d, const PalLayerNormTensors* t, void* stream) {
  using namespace pal;
  LayerNormArgs A{};
  if (int rc = layer_norm_args(d, A)) return rc;
  if (!t || !t->x || !t->weight || !t->y) return PAL_E_NULL;
  if (!t->residual_out && (t->residual || d->drop.p > 0.0 || d->res_dtype != d->dtype)) return PAL_E_NULL;
  if ((uintptr_t)t->stats & 7) return PAL_E_ALIGN;
  A.x = t->x; A.res = t->residual; A.weight = t->weight; A.bias = t->bias; A.s = t->residual_out; A.y = t->y; A.stats = t->stats;
  layer_norm_dispatch<false>(d, A, (hipStream_t)stream);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

extern "C" size_t pal_layer_norm_bwd_workspace_bytes(const PalLayerNormDims* d) {
  using namespace pal;
  LayerNormArgs A{};
  if (layer_norm_args(d, A) != PAL_OK) return 0;
  return sizeof(float) * (size_t)layer_norm_blocks(d->rows, d->dim, true) * 2 * d->dim;
}

extern "C" int pal_layer_norm_bwd(const PalLayerNormDims* d, const PalLayerNormTensors* t, const PalLayerNormGrads* gr, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace pal;
  LayerNormArgs A{};
  if (int rc = layer_norm_args(d, A)) return rc;
  if (!t || !t->weight || !t->stats || (!t->residual_out && !t->x) || !gr || !gr->dx || !gr->dweight) return PAL_E_NULL;
  if (!t->residual_out && (d->drop.p > 0.0 || d->res_dtype != d->dtype)) return PAL_E_NULL;
  if (!t->bias != !gr->dbias) return PAL_E_NULL;
  if ((uintptr_t)t->stats & 7) return PAL_E_ALIGN;
  if (!workspace || workspace_bytes < pal_layer_norm_bwd_workspace_bytes(d)) return PAL_E_WORKSPACE;
  if (!is_aligned16(workspace)) return PAL_E_ALIGN;
  A.x = t->x; A.weight = t->weight; A.s = t->residual_out; A.stats = t->stats;
  A.dy = gr->dy; A.dres = gr->dresidual_out; A.dx = gr->dx; A.ds = gr->dresidual;
  A.part = (float*)workspace; A.dweight = gr->dweight; A.dbias = gr->dbias;
  hipStream_t s = (hipStream_t)stream;
  layer_norm_dispatch<true>(d, A, s);
  PAL_HIP_LAUNCH_CHECK();
  PAL_TIMED_LAUNCH(kKernLayerNormReduce, s, layer_norm_reduce_kernel, dim3((2 * d->dim + 15) / 16), dim3(1024), 0, s, A.part, A.dweight, A.dbias,
                   layer_norm_blocks(d->rows, d->dim, true), d->dim);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

extern "C" int pal_dropout(const PalDropout* drop, const void* x, void* y, int64_t rows, int64_t dim, int64_t x_stride, int32_t dtype,
                           void* stream) {
  using namespace pal;
  if (!drop || !x || !y) return PAL_E_NULL;
  if (dtype != PAL_DTYPE_F32 && dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (rows <= 0 || dim <= 0 || dim > (int64_t)1 << 30 || rows > (int64_t)1 << 40 || x_stride < dim) return PAL_E_DIM;
  DropoutArgs A{};
  if (int rc = drop_args(*drop, A.drop)) return rc;
  A.x = x; A.y = y; A.stride = x_stride; A.dim = (uint32_t)dim;
  A.per_row = (uint32_t)((dim + 7) / 8);
  if (rows > ((int64_t)1 << 43) / A.per_row) return PAL_E_DIM;
  A.pieces = rows * A.per_row;
  A.magic = (uint32_t)((((uint64_t)1 << 32) + A.per_row - 1) / A.per_row);
  const int64_t each = A.pieces / (256 * 2048);
  A.turns = each < 1 ? 1 : each > 2 ? 2 : (int)each;
  const int64_t blocks = (A.pieces + 256 * A.turns - 1) / (256 * A.turns);
  if (blocks > 1 << 23) A.turns = (int)((A.pieces + ((int64_t)256 << 23) - 1) / ((int64_t)256 << 23));   // threads of a launch: more turns
  const dim3 grid((unsigned)((A.pieces + (int64_t)256 * A.turns - 1) / ((int64_t)256 * A.turns)));
  if (dtype == PAL_DTYPE_BF16) PAL_TIMED_LAUNCH(kKernDropout, (hipStream_t)stream, dropout_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, A);
  else PAL_TIMED_LAUNCH(kKernDropout, (hipStream_t)stream, dropout_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, A);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
