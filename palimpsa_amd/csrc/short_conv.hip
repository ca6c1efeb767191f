// Short causal convolution, one filter of `width` taps per channel, with its activation and its state:
//     p[t,c] = bias[c] + sum_{i<W} w[c, W-1-i] x[t-i,c],    y = p  or  p sigmoid(p),
// x before the first token of a sequence taken from the state it starts with (column W + t of [N,D,W]), or zero.
// Backward, with dp = dy act'(p):  dx[t] = sum_i w[W-1-i] dp[t+i] (the tokens of the sequence),  dw[W-1-i] = sum_t dp[t] x[t-i],
// dbias = sum_t dp[t]; the state's gradient is dx at t < 0.
//
// Bound by HBM: a thread owns a few neighbouring channels of a run of tokens of one sequence and walks the run with the last
// inputs in registers, so a row is read once (and its last W - 1 tokens once more by the run after it).  Dense batches are cut into
// runs of equal length; packed ones take the tiles of the chunk table (64 tokens of one sequence at most), cut the same way, so
// that no thread looks for its sequence.  Partial sums of dw and dbias are added over the runs of a workgroup, then over the
// workgroups, in a fixed order.
#include "pal_common.h"
#include "pal_host.h"
#include "pal_profile.h"
#include "rows8.h"

namespace pal {

struct ConvArgs {
  const void *x, *weight, *bias, *init, *dy, *d_final;
  void *y, *final_, *dx, *d_init;
  const int32_t *cu, *table;
  float *part, *dweight, *dbias;
  int64_t xb, xt;          // strides of x
  int32_t T, D, N, chunks, weight_bf16, silu;
  int32_t run, runs;       // tokens per run, runs of the pass
  int32_t pieces;          // pieces of channels
  int32_t blocks;          // workgroups that convolve; the ones behind them write states
  int32_t per_tile;        // runs per tile of the table (packed), or per batch row
};

// run r: its sequence, the tokens [t0, t1) it covers and those of the sequence, [s0, s1), all counted in rows of the tensors
struct ConvRun {
  int32_t seq;
  int64_t t0, t1, s0, s1, row0;   // row0: first token of the batch row
  __device__ __forceinline__ ConvRun(const ConvArgs& a, int r) {
    const int tile = r / a.per_tile, sub = r - tile * a.per_tile;
    if (a.cu) {
      const int32_t* e = a.table + 4 * (int64_t)tile;
      seq = min(max(e[0], 0), a.N - 1);
      int bos, len;
      packed_seq_bounds(a.cu, seq, a.T, bos, len);
      s0 = bos;
      s1 = (int64_t)bos + len;
      row0 = 0;
      const int64_t first = min(max((int64_t)e[1], s0), s1), last = min(first + min(max(e[2], 0), PAL_CHUNK), s1);
      t0 = min(first + (int64_t)sub * a.run, last);
      t1 = min(t0 + a.run, last);
    } else {
      seq = tile;
      s0 = row0 = (int64_t)tile * a.T;
      s1 = s0 + a.T;
      t0 = s0 + (int64_t)sub * a.run;
      t1 = min(t0 + a.run, s1);
    }
  }
  // element of x at token t (a row of this run's batch row)
  __device__ __forceinline__ int64_t at(const ConvArgs& a, int64_t t) const {
    return a.cu ? t * a.xt : (int64_t)seq * a.xb + (t - row0) * a.xt;
  }
};

// VW neighbouring channels as fetched: eight of bf16 rows in the forward, four elsewhere (eight would leave the backward two
// waves a SIMD), one where there are fewer channels than that.  The last piece of a row whose channels are no multiple of VW is moved back
// to be whole: its first channels are computed twice, and written twice with the same values.
template <typename T, int VW>
struct Chans;
template <typename T>
struct Chans<T, 8> {
  Piece8<T> v;
  __device__ __forceinline__ void load(const T* p) { v.load(p); }
  __device__ __forceinline__ float get(int e) const { return v.get(e); }
};
template <>
struct Chans<bf16_t, 4> {
  typedef bf16x4 any __attribute__((aligned(2)));
  bf16x4 v;
  __device__ __forceinline__ void load(const bf16_t* p) { v = *(const any*)p; }
  __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
};
template <>
struct Chans<float, 4> {
  f32x4 v;
  __device__ __forceinline__ void load(const float* p) { v = *(const f32x4_any*)p; }
  __device__ __forceinline__ float get(int e) const { return v[e]; }
};
template <typename T>
struct Chans<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ float get(int) const { return to_f32(v); }
};
template <int VW>
__device__ __forceinline__ void store_chans(bf16_t* p, const float* x) {
  if constexpr (VW == 8) {
    store_piece(p, x, 8);
  } else if constexpr (VW == 4) {
    typedef bf16x4 any __attribute__((aligned(2)));
    const bf16x2 a = pack2(x[0], x[1]), b = pack2(x[2], x[3]);
    const bf16x4 v = {a[0], a[1], b[0], b[1]};
    *(any*)p = v;
  } else {
    *p = (bf16_t)x[0];
  }
}
template <int VW>
__device__ __forceinline__ void store_chans(float* p, const float* x) {
  if constexpr (VW == 4) {
    const f32x4 v = {x[0], x[1], x[2], x[3]};
    *(f32x4_any*)p = v;
  } else {
    *p = x[0];
  }
}

// n consecutive parameters of either type; whichever it is, they are waited for in their branch (where the two meet, the compiler
// would wait for everything in flight)
template <int N>
__device__ __forceinline__ void load_run(float* x, const void* p, int64_t i, int is_bf16) {
  if (is_bf16) {
    const bf16_t* q = (const bf16_t*)p + i;
    if constexpr (N % 4 == 0) {
      typedef bf16x4 any __attribute__((aligned(2)));
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const bf16x4 v = *(const any*)(q + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k + e] = (float)v[e];
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = (float)q[k];
    }
  } else {
    const float* q = (const float*)p + i;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const f32x4 v = *(const f32x4_any*)(q + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k + e] = v[e];
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = q[k];
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) asm volatile("" : "+v"(x[k]));
}
template <int W, int VW>
__device__ __forceinline__ void load_taps(float (*w)[VW], float* bias, const ConvArgs& a, int c) {
  float x[VW * W];
  load_run<VW * W>(x, a.weight, (int64_t)c * W, a.weight_bf16);
#pragma unroll
  for (int e = 0; e < VW; ++e) {
    bias[e] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][e] = x[e * W + k];
  }
  if (a.bias) load_run<VW>(bias, a.bias, c, a.weight_bf16);
}
// the W - 1 inputs before the run: rows of the sequence, or the state it starts with, or zero; h[0] the oldest.  A run that is not the
// first of its sequence has a whole run before it, at least 8 tokens; where a table that was not made from these bounds says otherwise, the rows
// before the sequence (of the first one: before the tensor) are not read.
template <typename T, int W, int VW>
__device__ __forceinline__ void load_before(float (*h)[VW], const ConvArgs& a, const ConvRun& r, int c) {
  if (r.t0 - r.s0 >= W - 1) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      Chans<T, VW> x;
      x.load((const T*)a.x + r.at(a, r.t0 - (W - 1) + k) + c);
#pragma unroll
      for (int e = 0; e < VW; ++e) h[k][e] = x.get(e);
    }
  } else {
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
      for (int e = 0; e < VW; ++e) h[k][e] = a.init ? to_f32(((const T*)a.init)[((int64_t)r.seq * a.D + c + e) * W + k + 1]) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
#pragma unroll
    for (int e = 0; e < VW; ++e) asm volatile("" : "+v"(h[k][e]));
}

// final states: the last W inputs of a sequence, its old state moved up where it is shorter
template <typename T>
__device__ __forceinline__ void conv_states(const ConvArgs& a, int W, int block) {
  const int64_t total = (int64_t)a.N * a.D * W;
  for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < total; i += (int64_t)(gridDim.x - a.blocks) * 256) {
    const int k = (int)(i % W);
    const int64_t nc = i / W;
    const int c = (int)(nc % a.D), seq = (int)(nc / a.D);
    int64_t s0 = (int64_t)seq * a.T, len = a.T;
    if (a.cu) {
      int bos, l;
      packed_seq_bounds(a.cu, seq, a.T, bos, l);
      s0 = bos;
      len = l;
    }
    const int64_t t = len - W + k;
    T v = (T)0.f;
    if (t >= 0) v = ((const T*)a.x)[(a.cu ? (s0 + t) * a.xt : (int64_t)seq * a.xb + t * a.xt) + c];
    else if (a.init) v = ((const T*)a.init)[nc * W + k + len];
    ((T*)a.final_)[i] = v;
  }
}

constexpr int kConvBatch = 4;   // rows fetched together, one batch ahead

template <typename T, int W, int VW>
__global__ __launch_bounds__(256) void short_conv_fwd_kernel(ConvArgs a) {
  if ((int)blockIdx.x >= a.blocks) {
    conv_states<T>(a, W, blockIdx.x - a.blocks);
    return;
  }
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const int run = idx / a.pieces, c = min((int)(idx - (unsigned)run * a.pieces) * VW, a.D - VW);
  if (run >= a.runs) return;
  const ConvRun r(a, run);
  if (r.t0 >= r.t1) return;
  const int len = (int)(r.t1 - r.t0);
  const T* px = (const T*)a.x + r.at(a, r.t0) + c;
  T* py = (T*)a.y + r.t0 * a.D + c;
  Chans<T, VW> xb[kConvBatch];
#pragma unroll
  for (int u = 0; u < kConvBatch; ++u) xb[u].load(px + (int64_t)min(u, len - 1) * a.xt);
  float w[W][VW], bias[VW], h[W][VW];
  load_taps<W, VW>(w, bias, a, c);
  load_before<T, W, VW>(h, a, r, c);
  auto one = [&](const Chans<T, VW>& x, T* to) {
    float p[VW];
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      h[W - 1][e] = x.get(e);
      p[e] = bias[e];
#pragma unroll
      for (int k = 0; k < W; ++k) p[e] = fmaf(w[k][e], h[k][e], p[e]);
#pragma unroll
      for (int k = 0; k < W - 1; ++k) h[k][e] = h[k + 1][e];
    }
    if (a.silu)
#pragma unroll
      for (int e = 0; e < VW; ++e) p[e] *= logistic(p[e]);
    store_chans<VW>(to, p);
  };
  int tb = 0;
  for (; tb + kConvBatch <= len; tb += kConvBatch) {
    Chans<T, VW> next[kConvBatch];
#pragma unroll
    for (int u = 0; u < kConvBatch; ++u) next[u].load(px + (int64_t)min(tb + kConvBatch + u, len - 1) * a.xt);
#pragma unroll
    for (int u = 0; u < kConvBatch; ++u) one(xb[u], py + (int64_t)(tb + u) * a.D);
#pragma unroll
    for (int u = 0; u < kConvBatch; ++u) xb[u] = next[u];
  }
#pragma unroll
  for (int u = 0; u < kConvBatch - 1; ++u)
    if (tb + u < len) one(xb[u], py + (int64_t)(tb + u) * a.D);
}

// workgroups: (group of 4 runs, 64 pieces of channels), the pieces of a group next to each other; a wave walks one run, the
// four waves' shares of dw and dbias meet in LDS
template <typename T, int W, int VW>
__global__ __launch_bounds__(256) void short_conv_bwd_kernel(ConvArgs a) {
  __shared__ __attribute__((aligned(16))) float sW[4][W + 1][64 * VW + 4];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int spans = (a.pieces + 63) / 64, group = blockIdx.x / spans, span = blockIdx.x - group * spans;
  const int piece = span * 64 + lane, c = min(piece * VW, a.D - VW);
  const int run = group * 4 + wave;
  float dw[W][VW], db[VW];
#pragma unroll
  for (int e = 0; e < VW; ++e) {
    db[e] = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][e] = 0.f;
  }
  if (run < a.runs && piece < a.pieces) {
    const ConvRun r(a, run);
    if (r.t0 < r.t1) {
      const T* px = (const T*)a.x + r.at(a, r.t0) + c;
      const T* pg = (const T*)a.dy + r.t0 * a.D + c;
      T* pd = (T*)a.dx + r.t0 * a.D + c;
      const int len = (int)(r.t1 - r.t0), left = (int)min(r.s1 - r.t0, (int64_t)len + W - 1);   // tokens to walk, past the run
      const bool first = r.t0 == r.s0;
      struct Pair {
        Chans<T, VW> x, g;
      };
      auto fetch = [&](Pair& b, int t) {
        const int64_t at = min(t, left - 1);
        b.x.load(px + at * a.xt);
        b.g.load(pg + at * a.D);
      };
      Pair pb[W - 1], mb[kConvBatch];
#pragma unroll
      for (int u = 0; u < W - 1; ++u) fetch(pb[u], u);
#pragma unroll
      for (int u = 0; u < kConvBatch; ++u) fetch(mb[u], W - 1 + u);
      float w[W][VW], bias[VW], h[W][VW], dp[W][VW];   // dp[k]: token t - (W - 1) + k
      load_taps<W, VW>(w, bias, a, c);
      load_before<T, W, VW>(h, a, r, c);
#pragma unroll
      for (int e = 0; e < VW; ++e)
#pragma unroll
        for (int k = 0; k < W; ++k) dp[k][e] = 0.f;
      // takes token t in; dx: the gradient of token t - (W - 1), which is whole now.  in: the token is one of the sequence; own: of the run
      auto one = [&](const Pair& b, bool in, bool own, float* dx) {
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          h[W - 1][e] = b.x.get(e);
          float p = bias[e];
#pragma unroll
          for (int k = 0; k < W; ++k) p = fmaf(w[k][e], h[k][e], p);
          float g = b.g.get(e);
          if (a.silu) {
            const float s = logistic(p);
            g *= s + p * s * (1.f - s);
          }
          g = in ? g : 0.f;
          dp[W - 1][e] = g;
          dx[e] = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k) dx[e] = fmaf(w[W - 1 - k][e], dp[k][e], dx[e]);
          const float go = own ? g : 0.f;
          db[e] += go;
#pragma unroll
          for (int k = 0; k < W; ++k) dw[k][e] = own ? fmaf(go, h[k][e], dw[k][e]) : dw[k][e];
#pragma unroll
          for (int k = 0; k < W - 1; ++k) { h[k][e] = h[k + 1][e]; dp[k][e] = dp[k + 1][e]; }
        }
      };
      // what came back through the final state, where token r.t0 + t is one of the last W
      auto with_final = [&](int t, float* dx) {
        const int64_t slot = r.t0 + t - r.s1 + W;
        if (a.d_final && slot >= 0)
#pragma unroll
          for (int e = 0; e < VW; ++e) {
            float d = to_f32(((const T*)a.d_final)[((int64_t)r.seq * a.D + c + e) * W + slot]);
            asm volatile("" : "+v"(d));
            dx[e] += d;
          }
      };
      float dx[VW];
#pragma unroll
      for (int t = 0; t < W - 1; ++t) {
        one(pb[t], t < left, t < len, dx);
        if (first && a.d_init) {     // the gradient of the state's input t + 1 (the oldest, 0, meets no tap)
          with_final(t - (W - 1), dx);
#pragma unroll
          for (int e = 0; e < VW; ++e) {
            T* d = (T*)a.d_init + ((int64_t)r.seq * a.D + c + e) * W;
            d[t + 1] = from_f32<T>(dx[e]);
            if (t == 0) d[0] = (T)0.f;
          }
        }
      }
      int tb = W - 1;
      for (; tb + kConvBatch <= len; tb += kConvBatch) {
        Pair next[kConvBatch];
#pragma unroll
        for (int u = 0; u < kConvBatch; ++u) fetch(next[u], tb + kConvBatch + u);
#pragma unroll
        for (int u = 0; u < kConvBatch; ++u) {
          one(mb[u], true, true, dx);
          with_final(tb + u - (W - 1), dx);
          store_chans<VW>(pd + (int64_t)(tb + u - (W - 1)) * a.D, dx);
        }
#pragma unroll
        for (int u = 0; u < kConvBatch; ++u) mb[u] = next[u];
      }
      // the last tokens of the run, and the W - 1 behind it
      for (; tb < len + W - 1; tb += kConvBatch) {
        Pair next[kConvBatch];
        if (tb + kConvBatch < len + W - 1)
#pragma unroll
          for (int u = 0; u < kConvBatch; ++u) fetch(next[u], tb + kConvBatch + u);
#pragma unroll
        for (int u = 0; u < kConvBatch; ++u) {
          const int t = tb + u;
          if (t >= len + W - 1) break;
          one(mb[u], t < left, t < len, dx);
          with_final(t - (W - 1), dx);
          store_chans<VW>(pd + (int64_t)(t - (W - 1)) * a.D, dx);
        }
#pragma unroll
        for (int u = 0; u < kConvBatch; ++u) mb[u] = next[u];
      }
    }
  }
#pragma unroll
  for (int k = 0; k <= W; ++k)
#pragma unroll
    for (int e = 0; e < VW; ++e) sW[wave][k][VW * lane + e] = k < W ? dw[k < W ? k : 0][e] : db[e];
  __syncthreads();
  for (int i = threadIdx.x; i < (W + 1) * 64 * VW; i += 256) {
    const int k = i / (64 * VW), cc = i - k * (64 * VW), pc = span * 64 + cc / VW;
    if (pc < a.pieces)
      a.part[((int64_t)group * (W + 1) + k) * a.D + min(pc * VW, a.D - VW) + cc % VW] = sW[0][k][cc] + sW[1][k][cc] + sW[2][k][cc] + sW[3][k][cc];
  }
}

// dweight [D,W], dbias [D] from the workgroups' shares [groups][W+1][D] (16 waves, each its share in order), and behind these
// workgroups the gradient of the state of sequences without a token: it went straight through
template <typename T>
__global__ __launch_bounds__(1024) void short_conv_reduce_kernel(ConvArgs a, int W, int groups, int sum_blocks) {
  __shared__ float s[16][64];
  if ((int)blockIdx.x >= sum_blocks) {
    const int64_t total = (int64_t)a.N * a.D * W;
    for (int64_t i = (int64_t)(blockIdx.x - sum_blocks) * 1024 + threadIdx.x; i < total; i += (int64_t)(gridDim.x - sum_blocks) * 1024) {
      int bos, len;
      packed_seq_bounds(a.cu, (int)(i / ((int64_t)a.D * W)), a.T, bos, len);
      if (len == 0) ((T*)a.d_init)[i] = a.d_final ? ((const T*)a.d_final)[i] : (T)0.f;
    }
    return;
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane, cols = (int64_t)(W + 1) * a.D;
  float t = 0.f;
  if (col < cols)
    for (int g = w; g < groups; g += 16) t += a.part[g * cols + col];
  s[w][lane] = t;
  __syncthreads();
  if (w == 0 && col < cols) {
    t = s[0][lane];
#pragma unroll
    for (int k = 1; k < 16; ++k) t += s[k][lane];
    const int k = (int)(col / a.D), c = (int)(col - (int64_t)k * a.D);
    if (k < W) a.dweight[(int64_t)c * W + k] = t;
    else if (a.dbias) a.dbias[c] = t;
  }
}

// a few tokens of a generation: thread = channel of a sequence, state in place
template <typename T, int W>
__global__ __launch_bounds__(256) void short_conv_step_kernel(ConvArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.N * a.D) return;
  const int seq = (int)(i / a.D), c = (int)(i - (int64_t)seq * a.D);
  T* st = (T*)a.final_ + i * W;
  T h[W];
  float w[W];
#pragma unroll
  for (int k = 0; k < W; ++k) { h[k] = st[k]; w[k] = load_rt(a.weight, (int64_t)c * W + k, a.weight_bf16); }
  const float bias = a.bias ? load_rt(a.bias, c, a.weight_bf16) : 0.f;
  const T* px = (const T*)a.x + (int64_t)seq * a.xb + c;
  T* py = (T*)a.y + (int64_t)seq * a.T * a.D + c;
  for (int t = 0; t < a.T; ++t) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) h[k] = h[k + 1];
    h[W - 1] = px[t * a.xt];
    float p = bias;
#pragma unroll
    for (int k = 0; k < W; ++k) p = fmaf(w[k], to_f32(h[k]), p);
    if (a.silu) p *= logistic(p);
    py[(int64_t)t * a.D] = from_f32<T>(p);
  }
#pragma unroll
  for (int k = 0; k < W; ++k) st[k] = h[k];
}

static int check_conv(const PalConvDims* d, const PalConvTensors* t) {
  if (!d || !t) return PAL_E_NULL;
  if (d->batch <= 0 || d->seq_len <= 0 || d->n_seqs <= 0 || d->channels <= 0) return PAL_E_DIM;
  if ((int64_t)d->batch * d->seq_len > (int64_t)1 << 30 || d->channels > 1 << 20) return PAL_E_DIM;
  if (d->width < 2 || d->width > PAL_CONV_MAX_WIDTH) return PAL_E_DIM;
  if (d->dtype != PAL_DTYPE_F32 && d->dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->weight_dtype != PAL_DTYPE_F32 && d->weight_dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->x_token_stride < d->channels && d->seq_len > 1) return PAL_E_DIM;
  if (d->x_batch_stride < 0) return PAL_E_DIM;
  if (!t->x || !t->weight || !t->y) return PAL_E_NULL;
  return PAL_OK;
}
static int check_conv_seqs(const PalConvDims* d, const PalConvTensors* t) {
  const bool packed = d->flags & PAL_FLAG_VARLEN;
  if (packed && d->batch != 1) return PAL_E_VARLEN_BATCH;
  if (packed != (t->cu_seqlens != nullptr)) return PAL_E_CU_SEQLENS;
  if (!packed && d->n_seqs != d->batch) return PAL_E_DIM;
  if (packed && !t->chunk_table) return PAL_E_NULL;
  if (packed) {
    const int64_t lo = ((int64_t)d->seq_len + PAL_CHUNK - 1) / PAL_CHUNK, hi = (int64_t)d->seq_len / PAL_CHUNK + d->n_seqs;
    if (d->total_chunks < lo || d->total_chunks > hi) return PAL_E_CHUNK;
  }
  if (((d->flags & PAL_FLAG_HAS_INIT) != 0) != (t->init != nullptr)) return PAL_E_STATE;
  return PAL_OK;
}

static ConvArgs conv_args(const PalConvDims* d, const PalConvTensors* t) {
  ConvArgs a{};
  a.x = t->x; a.weight = t->weight; a.bias = t->bias; a.init = t->init; a.y = t->y; a.final_ = t->final_;
  a.cu = t->cu_seqlens; a.table = t->chunk_table;
  a.xb = d->x_batch_stride; a.xt = d->x_token_stride;
  a.T = d->seq_len; a.D = d->channels; a.N = d->n_seqs; a.chunks = d->total_chunks;
  a.weight_bf16 = d->weight_dtype == PAL_DTYPE_BF16; a.silu = d->silu;
  return a;
}
// Tokens per run: 64, halved down to 8 while the pass has less than 16 waves a compute unit.  (16384 tokens of 1536 channels in documents of 20
// tokens, forward and backward: 65 us; by the tokens alone, with runs of 8 that mostly are empty, 110.)
static void conv_runs(ConvArgs& a, const PalConvDims* d, int vw) {
  a.pieces = (a.D + vw - 1) / vw;
  a.run = PAL_CHUNK;
  const int64_t tokens = a.cu ? (int64_t)PAL_CHUNK * a.chunks : (int64_t)d->batch * d->seq_len;   // (a tile counts as full: short documents
                                                                                                   // take one run each, not several empty ones)
  while (a.run > 8 && tokens / a.run * a.pieces < 256 * 16 * 64) a.run >>= 1;
  a.per_tile = a.cu ? PAL_CHUNK / a.run : (a.T + a.run - 1) / a.run;
  a.runs = a.per_tile * (a.cu ? a.chunks : d->batch);
}

// workgroups of 256 that one launch holds: below 2^32 threads
constexpr int64_t kConvMostBlocks = (int64_t)1 << 23;

// channels per thread
static int conv_piece(const PalConvDims* d, bool bwd) {
  const int vw = d->dtype == PAL_DTYPE_BF16 && !bwd ? 8 : 4;
  return d->channels >= vw ? vw : 1;
}
template <typename T, int VW>
static void conv_fwd_launch(const ConvArgs& a, int W, int grid, hipStream_t s) {
#define PAL_CONV(W_)                                                                                                     \
  case W_:                                                                                                               \
    PAL_TIMED_LAUNCH(kKernShortConvFwd, s, (short_conv_fwd_kernel<T, W_, VW>), dim3(grid), dim3(256), 0, s, a);           \
    break;
  switch (W) { PAL_CONV(2) PAL_CONV(3) PAL_CONV(4) PAL_CONV(5) PAL_CONV(6) PAL_CONV(7) PAL_CONV(8) }
#undef PAL_CONV
}
template <typename T, int VW>
static void conv_bwd_launch(const ConvArgs& a, int W, dim3 grid, hipStream_t s) {
#define PAL_CONV(W_)                                                                                            \
  case W_: PAL_TIMED_LAUNCH(kKernShortConvBwd, s, (short_conv_bwd_kernel<T, W_, VW>), grid, dim3(256), 0, s, a); break;
  switch (W) { PAL_CONV(2) PAL_CONV(3) PAL_CONV(4) PAL_CONV(5) PAL_CONV(6) PAL_CONV(7) PAL_CONV(8) }
#undef PAL_CONV
}
template <typename T>
static void conv_step_launch(const ConvArgs& a, int W, hipStream_t s) {
  const unsigned grid = (unsigned)(((int64_t)a.N * a.D + 255) / 256);
#define PAL_CONV(W_)                                                                                                  \
  case W_: PAL_TIMED_LAUNCH(kKernShortConvStep, s, (short_conv_step_kernel<T, W_>), dim3(grid), dim3(256), 0, s, a); break;
  switch (W) { PAL_CONV(2) PAL_CONV(3) PAL_CONV(4) PAL_CONV(5) PAL_CONV(6) PAL_CONV(7) PAL_CONV(8) }
#undef PAL_CONV
}
static int conv_state_blocks(const PalConvDims* d) {
  const int64_t b = ((int64_t)d->n_seqs * d->channels * d->width + 1023) / 1024;
  return (int)(b < 1024 ? b : 1024);
}
// runs of the backward pass and the groups of four whose shares it leaves
static int conv_groups(const ConvArgs& a) { return (a.runs + 3) / 4; }

}  // namespace pal

extern "C" int pal_short_conv_fwd(const PalConvDims* d, const PalConvTensors* t, void* stream) {
  using namespace pal;
  if (int rc = check_conv(d, t)) return rc;
  if (int rc = check_conv_seqs(d, t)) return rc;
  if (((d->flags & PAL_FLAG_STORE_FINAL) != 0) != (t->final_ != nullptr)) return PAL_E_STATE;
  if (t->final_ && t->final_ == t->init) return PAL_E_STATE;   // read by one workgroup, written by another
  ConvArgs a = conv_args(d, t);
  const int vw = conv_piece(d, false);
  conv_runs(a, d, vw);
  const int64_t blocks = ((int64_t)a.runs * a.pieces + 255) / 256;
  if (blocks > kConvMostBlocks) return PAL_E_DIM;
  a.blocks = (int)blocks;
  const int grid = a.blocks + (t->final_ ? conv_state_blocks(d) : 0);
  hipStream_t s = (hipStream_t)stream;
  if (d->dtype == PAL_DTYPE_BF16) vw == 8 ? conv_fwd_launch<bf16_t, 8>(a, d->width, grid, s) : conv_fwd_launch<bf16_t, 1>(a, d->width, grid, s);
  else vw == 4 ? conv_fwd_launch<float, 4>(a, d->width, grid, s) : conv_fwd_launch<float, 1>(a, d->width, grid, s);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

extern "C" size_t pal_short_conv_bwd_workspace_bytes(const PalConvDims* d) {
  using namespace pal;
  PalConvTensors any{};
  any.x = any.weight = d; any.y = (void*)d;
  if (check_conv(d, &any) != PAL_OK) return 0;
  if (d->flags & PAL_FLAG_VARLEN) any.cu_seqlens = (const int32_t*)d;
  ConvArgs a = conv_args(d, &any);
  conv_runs(a, d, conv_piece(d, true));
  return sizeof(float) * (size_t)conv_groups(a) * (d->width + 1) * d->channels;
}

extern "C" int pal_short_conv_bwd(const PalConvDims* d, const PalConvTensors* t, const PalConvGrads* gr, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace pal;
  if (int rc = check_conv(d, t)) return rc;
  if (int rc = check_conv_seqs(d, t)) return rc;
  if (!gr || !gr->dy || !gr->dx || !gr->dweight || (t->bias != nullptr) != (gr->dbias != nullptr)) return PAL_E_NULL;
  if (gr->d_init && !t->init) return PAL_E_STATE;
  if (!workspace || workspace_bytes < pal_short_conv_bwd_workspace_bytes(d)) return PAL_E_WORKSPACE;
  ConvArgs a = conv_args(d, t);
  const int vw = conv_piece(d, true);
  conv_runs(a, d, vw);
  a.dy = gr->dy; a.dx = gr->dx; a.dweight = gr->dweight; a.dbias = gr->dbias; a.d_init = gr->d_init; a.d_final = gr->d_final;
  a.part = (float*)workspace;
  const int groups = conv_groups(a);
  const int64_t blocks = (int64_t)((a.pieces + 63) / 64) * groups;
  if (blocks > kConvMostBlocks) return PAL_E_DIM;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks);
  if (d->dtype == PAL_DTYPE_BF16) vw == 4 ? conv_bwd_launch<bf16_t, 4>(a, d->width, grid, s) : conv_bwd_launch<bf16_t, 1>(a, d->width, grid, s);
  else vw == 4 ? conv_bwd_launch<float, 4>(a, d->width, grid, s) : conv_bwd_launch<float, 1>(a, d->width, grid, s);
  PAL_HIP_LAUNCH_CHECK();
  const int sums = (int)(((int64_t)(d->width + 1) * a.D + 63) / 64), more = a.cu && a.d_init ? conv_state_blocks(d) : 0;
  if (d->dtype == PAL_DTYPE_BF16)
    PAL_TIMED_LAUNCH(kKernShortConvReduce, s, short_conv_reduce_kernel<bf16_t>, dim3(sums + more), dim3(1024), 0, s, a, d->width, groups, sums);
  else
    PAL_TIMED_LAUNCH(kKernShortConvReduce, s, short_conv_reduce_kernel<float>, dim3(sums + more), dim3(1024), 0, s, a, d->width, groups, sums);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}

extern "C" int pal_short_conv_step(const PalConvDims* d, const PalConvTensors* t, void* stream) {
  using namespace pal;
  if (int rc = check_conv(d, t)) return rc;
  if (d->flags & PAL_FLAG_VARLEN) return PAL_E_VARLEN_BATCH;
  if (d->n_seqs != d->batch) return PAL_E_DIM;
  if (!t->final_) return PAL_E_STATE;
  if ((int64_t)d->n_seqs * d->channels > 256 * kConvMostBlocks) return PAL_E_DIM;
  ConvArgs a = conv_args(d, t);
  if (d->dtype == PAL_DTYPE_BF16) conv_step_launch<bf16_t>(a, d->width, (hipStream_t)stream);
  else conv_step_launch<float>(a, d->width, (hipStream_t)stream);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
