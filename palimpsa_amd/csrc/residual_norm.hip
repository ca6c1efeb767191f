// Pre-norm of a residual block with the addition in front of it:
//     s = x + residual (rounded to the residual stream's type, handed on),   y = s r w,   r = 1 / sqrt(mean s^2 + eps)
// with rows of y in the type of x, or in 8 bits (OCP e4m3) with one fp32 scale per row or per group of the row:
//     scale = max(max |y|, 1e-12) / 448,   q = round(y / scale).
// Backward, with dy and the gradient dres that comes back along the stream (both may be missing):
//     ds = r (w dy - s r mean(w dy s r)) + dres  (the gradient of x and of residual),   dw = sum over rows of dy s r.
// It reads s as the forward call handed it on and takes the mean square again, so nothing else is kept between the two.
//
// Bound by HBM: every row is read once and written once.  A row is held in registers by one wave (up to 2048 entries) or by
// the four waves of a workgroup (up to 16384), eight neighbouring entries per lane and piece; a wave walks several rows with the
// weights in registers and fetches the next row before it sums the present one.  16384 rows of 1536, bf16 beside an fp32 stream: forward 302 MB
// in 58 us, backward 403 MB in 71; 16384 rows of 2048 to 8 bits with groups of 128: 235 MB in 44 us.
#include "pal_common.h"
#include "pal_host.h"
#include "pal_profile.h"
#include "rows8.h"

namespace pal {

constexpr float kFp8Max = 448.f, kFp8Least = 1e-12f;   // largest e4m3 number; |y| below the second counts as that much
constexpr int kNormMaxRow = 16384;

struct NormArgs {
  const void *x, *res, *weight;
  void *res_out, *y;
  float* scales;
  const void *dy, *dres;
  void *dx, *dres_in;     // dres_in: the same gradient in the type of the residual stream (NULL: the types are one)
  float *part, *dweight;  // [workgroups][dim]; [dim]
  int64_t rows;
  int64_t x_stride, res_stride;   // elements between rows of x and of residual (all other rows are packed)
  int dim, weight_bf16, group;
  float eps;
};

// sum over the waves of a row; `turn` alternates between two slots so that one barrier per sum is enough
template <int WPR>
__device__ __forceinline__ float row_sum(float x, float (*s)[4], int turn) {
  x = wave_sum(x);
  if constexpr (WPR > 1) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) s[turn][w] = x;
    __syncthreads();
    x = s[turn][0] + s[turn][1] + s[turn][2] + s[turn][3];
  }
  return x;
}
template <int WPR>
__device__ __forceinline__ float row_max(float x, float (*s)[4], int turn) {
  x = wave_max(x);
  if constexpr (WPR > 1) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) s[turn][w] = x;
    __syncthreads();
    x = fmaxf(fmaxf(s[turn][0], s[turn][1]), fmaxf(s[turn][2], s[turn][3]));
  }
  return x;
}
// maximum over the lanes / 8 neighbours that hold a group (4 to 32 of them); every one gets it
template <int CTRL>
__device__ __forceinline__ float dpp_max(float x) {
  return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float group_max(float x, int lanes) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  if (lanes > 4) x = dpp_max<0x141>(x);   // row_half_mirror
  if (lanes > 8) x = dpp_max<0x140>(x);   // row_mirror
  if (lanes > 16) {
    float a = x, b = x;
    swap_rows(a, b);
    x = fmaxf(a, b);
  }
  return x;
}

// Piece v of a lane: eight entries from column `at` on.  Rows of eight entries or more, WHOLE: the last piece of a row whose length is no
// multiple of eight, and those of lanes behind it, are moved back to be whole, so that no load waits on a branch; what is there twice has
// the same values, is written twice and counts once in sums (entries from `from` on).  Shorter rows are read element by element.
template <int NV, int WPR, bool WHOLE>
struct NormPiece {
  int at, from;
  bool on;               // the lane has entries of its own
  __device__ __forceinline__ NormPiece(int lane, int v, int D) {
    const int c = 8 * (lane + 64 * WPR * v);
    on = c < D;
    at = WHOLE ? min(c, D - 8) : c;
    from = c - at;
  }
  // (one wave a row: all pieces but the last are whole)
  static constexpr bool masked(int v) { return WHOLE && (WPR > 1 || v == NV - 1); }
};
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_row_piece(Piece8<T>& d, const T* row, int at, int D) {
  if constexpr (WHOLE) d.load(row + at);
  else load_piece(d, row + at, D - at);
}

template <typename TX, typename TR, int NV, int WPR, bool FP8, bool WHOLE>
__global__ __launch_bounds__(256) void residual_norm_fwd_kernel(NormArgs A) {
  typedef NormPiece<NV, WPR, WHOLE> At;
  __shared__ float sSum[2][4], sMax[2][4];
  constexpr int kSlots = 4 / WPR, kStep = 64 * WPR;
  const int slot = WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
  const int lane = threadIdx.x & (kStep - 1);
  const int D = A.dim;
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kSlots;
  int64_t row = (int64_t)blockIdx.x * kSlots + slot;
  if (WPR == 1 && row >= A.rows) return;
  float w[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if constexpr (WHOLE) load_params(w[v], A.weight, At(lane, v, D).at, A.weight_bf16);
    else load_few_params(w[v], A.weight, A.weight_bf16, lane ? 0 : D);
  }
  Piece8<TX> xb[NV];
  Piece8<TR> rb[NV];
  const bool has_res = A.res != nullptr;
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      load_row_piece<WHOLE>(xb[v], (const TX*)A.x + r * A.x_stride, p.at, D);
      if (has_res) load_row_piece<WHOLE>(rb[v], (const TR*)A.res + r * A.res_stride, p.at, D);
    }
  };
  fetch(row);
  for (int turn = 0; row < A.rows; row += step, turn ^= 1) {
    float s[NV][8], ss = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[v][e] = has_res ? xb[v].get(e) + rb[v].get(e) : xb[v].get(e);
      if (p.on) store_piece((TR*)A.res_out + row * D + p.at, s[v], WHOLE ? 8 : D - p.at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[v][e] = to_f32(from_f32<TR>(s[v][e]));   // the norm is that of the stream as it is handed on
        const float q = fmaf(s[v][e], s[v][e], ss);
        ss = At::masked(v) && e < p.from ? ss : q;
      }
    }
    if (row + step < A.rows) fetch(row + step);
    ss = row_sum<WPR>(ss, sSum, turn);
    const float r = rsqrtf(fmaf(ss, inv_d, A.eps));
    if constexpr (!FP8) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const At p(lane, v, D);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = s[v][e] * r * w[v][e];
        if (p.on) store_piece((TX*)A.y + row * D + p.at, y, WHOLE ? 8 : D - p.at);
      }
    } else {
      float top[NV], all = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        top[v] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[v][e] *= r * w[v][e];
          top[v] = fmaxf(top[v], fabsf(s[v][e]));
        }
        all = fmaxf(all, top[v]);
      }
      const int groups = A.group ? D / A.group : 1;
      if (A.group) {
#pragma unroll
        for (int v = 0; v < NV; ++v) top[v] = group_max(top[v], A.group >> 3);
      } else {
        all = row_max<WPR>(all, sMax, turn);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const At p(lane, v, D);
        const int c = 8 * (lane + kStep * v);
        const float scale = fmaxf(A.group ? top[v] : all, kFp8Least) * (1.f / kFp8Max);
        // a row whose sum of squares is no finite number has NaN for its scales (the maximum above drops a NaN, the sum does not)
        const float sc = r > 0.f ? scale : __builtin_nanf("");
        const float inv = 1.f / sc;
        if (p.on) {
          if (A.group ? (c & (A.group - 1)) == 0 : c == 0) A.scales[row * groups + (A.group ? c / A.group : 0)] = sc;
          int q[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // at most 448 and a few roundings in absolute value, which the conversion rounds to 448: no clamp is needed
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = s[v][4 * h + e] * inv;
            q[h] = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
            q[h] = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], q[h], true);
          }
          unsigned char* out = (unsigned char*)A.y + row * D + p.at;
          if (WHOLE || D >= 8) {
            typedef int i32x2_any __attribute__((ext_vector_type(2), aligned(1)));
            i32x2_any o = {q[0], q[1]};
            *(i32x2_any*)out = o;
          } else {
            for (int e = 0; e < D; ++e) out[e] = (unsigned char)(q[e >> 2] >> (8 * (e & 3)));
          }
        }
      }
    }
  }
}

// (two waves a SIMD where a row of 1536 entries or less is all that a wave holds)
template <typename TX, typename TR, int NV, int WPR, bool WHOLE>
__global__ __launch_bounds__(256, WPR == 1 && NV <= 3 ? 2 : 1) void residual_norm_bwd_kernel(NormArgs A) {
  typedef NormPiece<NV, WPR, WHOLE> At;
  __shared__ float sSum[2][4], sDot[2][4];
  extern __shared__ float sW[];   // WPR == 1: [4 waves][512 NV] shares of dweight
  constexpr int kSlots = 4 / WPR, kStep = 64 * WPR;
  const int slot = WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
  const int lane = threadIdx.x & (kStep - 1);
  const int D = A.dim;
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kSlots;
  const bool has_dy = A.dy != nullptr, has_dres = A.dres != nullptr;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if constexpr (WHOLE) load_params(w[v], A.weight, At(lane, v, D).at, A.weight_bf16);
    else load_few_params(w[v], A.weight, A.weight_bf16, lane ? 0 : D);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[v][e] = 0.f;
  }
  Piece8<TR> sb[NV], eb[NV];
  Piece8<TX> gb[NV];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      load_row_piece<WHOLE>(sb[v], (const TR*)A.res_out + r * D, p.at, D);
      if (has_dy) load_row_piece<WHOLE>(gb[v], (const TX*)A.dy + r * D, p.at, D);
      if (has_dres) load_row_piece<WHOLE>(eb[v], (const TR*)A.dres + r * D, p.at, D);
    }
  };
  int64_t row = (int64_t)blockIdx.x * kSlots + slot;
  if (row < A.rows) fetch(row);
  for (int turn = 0; row < A.rows; row += step, turn ^= 1) {
    float s[NV][8], g[NV][8], ex[NV][8], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[v][e] = sb[v].get(e);
        g[v][e] = has_dy ? gb[v].get(e) : 0.f;
        ex[v][e] = has_dres ? eb[v].get(e) : 0.f;
        const float q = fmaf(s[v][e], s[v][e], ss), d = fmaf(g[v][e] * w[v][e], s[v][e], dot);
        const bool twice = At::masked(v) && e < p.from;
        ss = twice ? ss : q;
        dot = twice ? dot : d;
      }
    }
    if (row + step < A.rows) fetch(row + step);
    ss = row_sum<WPR>(ss, sSum, turn);
    dot = row_sum<WPR>(dot, sDot, turn);
    const float r = rsqrtf(fmaf(ss, inv_d, A.eps));
    // (never the cube of r by itself: it passes the range of fp32 for rows whose entries are beyond 1e13 or below 1e-13)
    const float mean = has_dy ? r * dot * inv_d : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[v][e] = fmaf(g[v][e] * r, s[v][e], dw[v][e]);
        d[e] = fmaf(r, fmaf(-s[v][e] * r, mean, g[v][e] * w[v][e]), ex[v][e]);
      }
      if (p.on) store_piece((TX*)A.dx + row * D + p.at, d, WHOLE ? 8 : D - p.at);
      if (p.on && A.dres_in) store_piece((TR*)A.dres_in + row * D + p.at, d, WHOLE ? 8 : D - p.at);
    }
  }
  // dweight: the waves' shares in their order
  if constexpr (WPR == 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      if (p.on) store_piece(sW + slot * NV * 512 + p.at, dw[v], WHOLE ? 8 : D - p.at);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += 256) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) t += sW[k * NV * 512 + c];
      A.part[(int64_t)blockIdx.x * D + c] = t;
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const At p(lane, v, D);
      if (p.on) store_piece(A.part + (int64_t)blockIdx.x * D + p.at, dw[v], WHOLE ? 8 : D - p.at);
    }
  }
}

// dweight[c]: 64 groups of sixteen threads take sixteen columns, each group its share of the workgroups in order.  (Sixteen waves on 64
// columns were 24 workgroups for 1536 of them: 10.8 us.)
__global__ __launch_bounds__(1024) void residual_norm_reduce_kernel(const float* part, float* out, int n, int dim) {
  __shared__ float s[64][17];
  const int x = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
  float t = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int j = g; j < n; j += 64) t += part[(int64_t)j * dim + c];
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
  if (g == 0 && c < dim) {
    t = s[0][x];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += s[k][x];
    out[c] = t;
  }
}

// workgroups of a pass: as many as there are rows for, at most eight waves a SIMD (forward) or two (backward, where each leaves a
// share of dweight behind that has to be added)
static int norm_blocks(int64_t rows, int dim, bool bwd) {
  const int slots = dim > 2048 ? 1 : 4;
  const int64_t want = (rows + slots - 1) / slots, most = bwd ? 512 : 2048;
  return (int)(want < most ? want : most);
}

// one wave a row up to 2048 entries, four beyond; pieces of eight per lane: enough for the row
template <typename TX, typename TR, bool BWD, bool FP8>
static void norm_launch(const NormArgs& A, hipStream_t s) {
  const dim3 grid(norm_blocks(A.rows, A.dim, BWD));
  const bool wide = A.dim > 2048;
  const int nv = (A.dim + (wide ? 2047 : 511)) / (wide ? 2048 : 512);
#define PAL_NORM(NV, WPR, WHOLE)                                                                                      \
  do {                                                                                                             \
    if constexpr (BWD) {                                                                                           \
      const size_t lds = WPR == 1 ? (size_t)4 * 512 * NV * sizeof(float) : 0;                                      \
      PAL_TIMED_LAUNCH(kKernResidualNormBwd, s, (residual_norm_bwd_kernel<TX, TR, NV, WPR, WHOLE>), grid, dim3(256), lds, s, A); \
    } else {                                                                                                       \
      PAL_TIMED_LAUNCH(kKernResidualNormFwd, s, (residual_norm_fwd_kernel<TX, TR, NV, WPR, FP8, WHOLE>), grid, dim3(256), 0, s, A); \
    }                                                                                                              \
  } while (0)
  if (!wide) {
    if (A.dim < 8) PAL_NORM(1, 1, false);
    else if (nv == 1) PAL_NORM(1, 1, true);
    else if (nv == 2) PAL_NORM(2, 1, true);
    else if (nv == 3) PAL_NORM(3, 1, true);
    else PAL_NORM(4, 1, true);
  } else {
    if (nv <= 2) PAL_NORM(2, 4, true);
    else if (nv <= 4) PAL_NORM(4, 4, true);
    else PAL_NORM(8, 4, true);
  }
#undef PAL_NORM
}
template <bool BWD, bool FP8>
static void norm_dispatch(const PalNormDims* d, const NormArgs& A, hipStream_t s) {
  if (d->dtype == PAL_DTYPE_F32) norm_launch<float, float, BWD, FP8>(A, s);
  else if (d->res_dtype == PAL_DTYPE_F32) norm_launch<bf16_t, float, BWD, FP8>(A, s);
  else norm_launch<bf16_t, bf16_t, BWD, FP8>(A, s);
}

static int check_norm(const PalNormDims* d) {
  if (!d) return PAL_E_NULL;
  if (d->rows <= 0 || d->dim <= 0 || d->dim > kNormMaxRow || d->rows > (int64_t)1 << 40) return PAL_E_DIM;
  if (d->dtype != PAL_DTYPE_F32 && d->dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->res_dtype != PAL_DTYPE_F32 && d->res_dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->dtype == PAL_DTYPE_F32 && d->res_dtype != PAL_DTYPE_F32) return PAL_E_DTYPE;
  if (d->weight_dtype != PAL_DTYPE_F32 && d->weight_dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->group && (d->group < 32 || d->group > 256 || (d->group & (d->group - 1)) || d->dim % d->group)) return PAL_E_DIM;
  if (d->x_stride < d->dim || d->res_stride < d->dim) return PAL_E_DIM;
  if (!(d->eps >= 0.f)) return PAL_E_DIM;
  return PAL_OK;
}
static NormArgs norm_args(const PalNormDims* d) {
  NormArgs A{};
  A.rows = d->rows; A.dim = d->dim; A.weight_bf16 = d->weight_dtype == PAL_DTYPE_BF16; A.group = d->group; A.eps = d->eps;
  A.x_stride = d->x_stride; A.res_stride = d->res_stride;
  return A;
}

}  // namespace pal

extern "C" int pal_residual_norm_fwd(const PalNormDims* d, const PalNormTensors* t, void* stream) {
  using namespace pal;
  if (int rc = check_norm(d)) return rc;
  if (!t || !t->x || !t->weight || !t->residual_out || !t->y) return PAL_E_NULL;
  NormArgs A = norm_args(d);
  A.x = t->x; A.res = t->residual; A.weight = t->weight; A.res_out = t->residual_out; A.y = t->y; A.scales = t->scales;
  if (t->scales) norm_dispatch<false, true>(d, A, (hipStream_t)stream);
  else norm_dispatch<false, false>(d, A, (hipStream_t)stream);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

extern "C" size_t pal_residual_norm_bwd_workspace_bytes(const PalNormDims* d) {
  using namespace pal;
  if (check_norm(d) != PAL_OK) return 0;
  return sizeof(float) * (size_t)norm_blocks(d->rows, d->dim, true) * d->dim;
}

extern "C" int pal_residual_norm_bwd(const PalNormDims* d, const PalNormTensors* t, const PalNormGrads* gr, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace pal;
  if (int rc = check_norm(d)) return rc;
  if (!t || !t->weight || !t->residual_out || !gr || !gr->dx || !gr->dweight) return PAL_E_NULL;
  if (d->dtype != d->res_dtype && !gr->dresidual) return PAL_E_NULL;
  if (!workspace || workspace_bytes < pal_residual_norm_bwd_workspace_bytes(d)) return PAL_E_WORKSPACE;
  if (!is_aligned16(workspace)) return PAL_E_ALIGN;
  NormArgs A = norm_args(d);
  A.weight = t->weight; A.res_out = t->residual_out;
  A.dy = gr->dy; A.dres = gr->dresidual_out; A.dx = gr->dx; A.dres_in = gr->dresidual;
  A.part = (float*)workspace; A.dweight = gr->dweight;
  hipStream_t s = (hipStream_t)stream;
  norm_dispatch<true, false>(d, A, s);
  PAL_HIP_LAUNCH_CHECK();
  PAL_TIMED_LAUNCH(kKernResidualNormReduce, s, residual_norm_reduce_kernel, dim3((d->dim + 15) / 16), dim3(1024), 0, s, A.part,
                   A.dweight, norm_blocks(d->rows, d->dim, true), d->dim);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
