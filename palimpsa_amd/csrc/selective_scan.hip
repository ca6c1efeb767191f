// Selective scan: a linear recurrence with a decay of its own for every channel d and state entry n,
//     dt = softplus(delta + bias),   h[d,n] = exp(dt A[d,n]) h[d,n] + dt u[d] B[n],   y[d] = (sum_n C[n] h[d,n] + D u[d]) silu(z[d]).
// Backward, with Y = dy silu(z) and g the gradient of the state after a token (g = C Y + what comes back from the next token):
//     dC[n] = sum_d Y h,  dB[n] = sum_d g dt u,  du = dt sum_n g B + D Y,  ddt = sum_n g (a h') A + u sum_n g B,
//     dA = sum_t dt g (a h'),  dD = sum_t Y u,  dz = dy (sum_n C h + D u) silu'(z),  back to the token before: a g
// with a = exp(dt A), h' the state before the token.  No two entries share a decay, so nothing here is a matrix product.
//
// Bound by the issue of vector instructions: an entry and token take an exponential and four multiplications or fused
// multiply-adds forward (8.3 + 4 x 2.7 cycles a wave on this GPU), an exponential and fifteen backward.  The shape of a wave
// follows from that: 64 channels by 16 state entries, a lane 4 by 4 of them.  Sums over n are then three quarters in registers
// and the rest over the four lanes of a quad, sums over d (dB, dC) a quarter in registers and the rest over the sixteen quads; and
// what is done once per channel and token (softplus, silu, their derivatives, loads and stores) is one channel for each lane, handed
// to its quad by lane moves.  State sizes above 16 take one wave for each sixteen, which add their sums in LDS.
//
// Where the channels and sequences of a pass are too few waves, the tokens are cut into segments: a first kernel walks each
// segment from zero and leaves its last state and the sum of its dt (the decay over the segment is exp(A sum dt)), a second
// joins them to the states the segments start with, the third is the pass itself.  The backward does the same from the end.  In a packed
// batch segments know nothing of sequences: a token that starts a sequence takes that sequence's initial state in place of the
// state before it, and a segment that holds such a token lets nothing through.
//
// For the backward the forward keeps the state before every 16th token in fp32; the backward computes the 16 tokens again, four
// at a time, and keeps a and a h' of four tokens in registers.
#include "pal_common.h"
#include "pal_host.h"
#include "pal_profile.h"

namespace pal {

struct ScanArgs {
  const void *u, *delta, *z, *Bm, *Cm, *dy;
  const float *A, *D, *bias, *init, *d_final;
  void *y, *du, *ddelta, *dz, *dB, *dC;
  float *final_, *d_init, *ckpt, *dA, *dD, *dbias;
  float *seg_h, *seg_dt, *part_bc, *part_a, *part_c;
  int32_t *seg_cut;
  const int32_t* cu;
  int64_t ub, ut, db, dt, zb, zt, Bb, Bt, Cb, Ct;   // strides
  int32_t rows, T, seqs, D_, N, G, per_group, tiles_g, tiles, softplus, vec;
  int32_t seg, segs, ckpts;                          // tokens per segment (a multiple of PAL_SCAN_BLOCK), segments and kept states per row
};

// ------------------------------------------------------------------------------------------------ scalar functions
// exp(x) with the rounding of x log2(e) made up for: relative error of a few 2^-24 at any x (0 below -87, e^88 above 88)
__device__ __forceinline__ float exp_full(float x) {
  x = __builtin_amdgcn_fmed3f(x, -150.f, 88.f);
  const float t = x * kLog2e, r = fmaf(x, kLog2e, -t) + x * 1.925963033e-8f;
  const float e = fast_exp2(t);
  return fmaf(e, r * 0.6931471806f, e);
}
// log(1 + e) for e >= 0: the rounding of 1 + e is made up for
__device__ __forceinline__ float log1p_full(float e) {
  const float s = 1.f + e;
  return fmaf(e - (s - 1.f), fast_rcp(s), __builtin_amdgcn_logf(s) * 0.6931471806f);
}
// time step from the raw one (already with its bias); softplus is the identity above 20, as torch computes it
__device__ __forceinline__ float time_step(float raw, int softplus) {
  return softplus && raw <= 20.f ? log1p_full(exp_full(raw)) : raw;
}
__device__ __forceinline__ float sigmoid_full(float x) { return fast_rcp(1.f + exp_full(-x)); }

// ------------------------------------------------------------------------------------------------ lanes
// lane 4 q + j of a wave: channels 16 k + q (k = 0 .. 3) by entries 4 j + i (i = 0 .. 3) of the state; its own channel is 16 j + q
template <int K>
__device__ __forceinline__ float of_channel(float x) { return quad_move<K * 0x55>(x); }   // the value of the lane that owns channel k
// four sums over a quad: lane j gets the total of p_j
__device__ __forceinline__ float quad_total4(float p0, float p1, float p2, float p3, bool odd, bool high) {
  const float a = (odd ? p1 : p0) + quad_move<0xB1>(odd ? p0 : p1);
  const float b = (odd ? p3 : p2) + quad_move<0xB1>(odd ? p2 : p3);
  return (high ? b : a) + quad_move<0x4E>(high ? a : b);
}

// a sequence: its number and its tokens [s, e) in the row
struct ScanSeq {
  int n, s, e;
};
__device__ __forceinline__ ScanSeq seq_at(const ScanArgs& a, int row, int t) {
  if (!a.cu) return {row, 0, a.T};
  int lo = 0, hi = a.seqs - 1;      // last sequence that starts at t or before: it holds t if any does
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return {lo, a.cu[lo], a.cu[lo + 1]};
}

template <typename T>
struct Lane {
  int w, j, q, n0, own, row, tile, group;
  bool on, odd, high;
  int chan[4], valid[4];
  __device__ __forceinline__ Lane(const ScanArgs& a) {
    const int l = threadIdx.x & 63;
    w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    q = l >> 2; j = l & 3;
    odd = j & 1; high = j & 2;
    n0 = 16 * w + 4 * j;
    tile = blockIdx.x;
    row = blockIdx.z;
    group = tile / a.tiles_g;
    const int base = group * a.per_group + (tile - group * a.tiles_g) * 64, end = (group + 1) * a.per_group;
    own = base + 16 * j + q;
    on = own < end;
    own = min(own, end - 1);        // (lanes beyond the group compute its last channel again and store nothing)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      chan[k] = base + 16 * k + q;
      valid[k] = chan[k] < end;
      chan[k] = min(chan[k], end - 1);
    }
  }
  // the lane's 4 x 4 entries of a [.., channels, N] fp32 array, zero beyond N
  __device__ __forceinline__ void load(const ScanArgs& a, const float* p, float (*x)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* s = p + (int64_t)chan[k] * a.N + n0;
      if (a.vec && n0 < a.N) {
        const f32x4 v = *(const f32x4*)s;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[k][i] = n0 + i < a.N ? s[i] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(const ScanArgs& a, float* p, const float (*x)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!valid[k]) continue;
      float* d = p + (int64_t)chan[k] * a.N + n0;
      if (a.vec && n0 < a.N) {
        const f32x4 v = {x[k][0], x[k][1], x[k][2], x[k][3]};
        *(f32x4*)d = v;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n0 + i < a.N) d[i] = x[k][i];
      }
    }
  }
  __device__ __forceinline__ void store_zero(const ScanArgs& a, float* p) const {
    const float z[4][4] = {};
    store(a, p, z);
  }
  // four entries of B or C of a token as fetched (zero beyond N)
  __device__ __forceinline__ void fetch_bc(const ScanArgs& a, const void* base, int64_t at, int n, float* x) const {
    const T* p = (const T*)base + at + (int64_t)group * a.N + n;
    if constexpr (sizeof(T) == 2) {
      typedef bf16x4 any __attribute__((aligned(2)));
      if (n + 4 <= a.N) {
        const bf16x4 v = *(const any*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
        return;
      }
    } else {
      typedef f32x4 any __attribute__((aligned(4)));
      if (n + 4 <= a.N) {
        const f32x4 v = *(const any*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i];
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = n + i < a.N ? to_f32(p[i]) : 0.f;
  }
};
// index of a lane's four entries in an array of one float4 for each lane, channel piece and wave of every tile
__device__ __forceinline__ int64_t packed_at(int64_t slot, const ScanArgs& a, int tile, int nw, int w, int k) {
  return (((slot * a.tiles + tile) * nw + w) * 4 + k) * 64 + (threadIdx.x & 63);
}
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// a sequence's state where it starts
template <typename T>
__device__ __forceinline__ void start_state(const ScanArgs& a, const Lane<T>& ln, int seq, float (*h)[4]) {
  if (a.init) {
    ln.load(a, a.init + (int64_t)seq * a.D_ * a.N, h);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) h[k][i] = 0.f;
  }
}

// ------------------------------------------------------------------------------------------------ forward
constexpr int kScanTok = 8;   // tokens fetched together

// OUT: the pass itself.  Otherwise the walk of a segment from zero: its last state, the sum of its dt, and whether a sequence starts in it.
template <typename T, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW) void scan_fwd_kernel(ScanArgs a) {
  __shared__ float sBC[NW][kScanTok][2][16];
  __shared__ float sY[NW > 1 && OUT ? 2 : 1][NW > 1 && OUT ? NW : 1][kScanTok][64];
  const Lane<T> ln(a);
  const int l = threadIdx.x & 63, w = ln.w, row = ln.row;
  const int t0 = blockIdx.y * a.seg, t1 = min(a.T, t0 + a.seg);
  const float bias = a.bias ? a.bias[ln.own] : 0.f, Dc = a.D ? a.D[ln.own] : 0.f;
  float A2[4][4], h[4][4], dt_sum = 0.f;
  ln.load(a, a.A, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) { A2[k][i] *= kLog2e; h[k][i] = 0.f; }
  ScanSeq cur = seq_at(a, row, t0);
  int cut = 0;
  if (OUT && t0 > 0 && cur.s != t0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 v = ((const f32x4*)a.seg_h)[packed_at((int64_t)row * a.segs + blockIdx.y, a, ln.tile, NW, w, k)];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[k][i] = v[i];
    }
  }
  if (OUT && t0 == 0 && a.final_ && a.cu)
    for (int n = 0; n < cur.n; ++n) {   // sequences without a token before the first one
      float x[4][4];
      start_state(a, ln, n, x);
      ln.store(a, a.final_ + (int64_t)n * a.D_ * a.N, x);
    }
  const T* pu = (const T*)a.u + row * a.ub + ln.own;
  const T* pd = (const T*)a.delta + row * a.db + ln.own;
  const T* pz = a.z ? (const T*)a.z + row * a.zb + ln.own : nullptr;
  T* py = (T*)a.y + (int64_t)row * a.T * a.D_ + ln.own;

  T ur[kScanTok], dr[kScanTok], zr[kScanTok];
  float bc[4];
  auto fetch = [&](int tb) {
#pragma unroll
    for (int t = 0; t < kScanTok; ++t) {
      const int64_t at = min(tb + t, t1 - 1);
      ur[t] = pu[at * a.ut];
      dr[t] = pd[at * a.dt];
      if (OUT && a.z) zr[t] = pz[at * a.zt];
    }
    const int64_t at = min(tb + (l >> 3), t1 - 1);
    const bool c = l & 4;
    if (OUT || !c) ln.fetch_bc(a, c ? a.Cm : a.Bm, c ? row * a.Cb + at * a.Ct : row * a.Bb + at * a.Bt, 16 * w + 4 * (l & 3), bc);
  };
  fetch(t0);
  int turn = 0;
  for (int tb = t0; tb < t1; tb += kScanTok) {
    if (OUT && a.ckpt && (tb & (PAL_SCAN_BLOCK - 1)) == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 v = {h[k][0], h[k][1], h[k][2], h[k][3]};
        ((f32x4*)a.ckpt)[packed_at((int64_t)row * a.ckpts + tb / PAL_SCAN_BLOCK, a, ln.tile, NW, w, k)] = v;
      }
    }
    const int nt = min(kScanTok, t1 - tb);
    float dt[kScanTok], x[kScanTok], uv[kScanTok], zv[kScanTok];
#pragma unroll
    for (int t = 0; t < kScanTok; ++t) {
      uv[t] = to_f32(ur[t]);
      dt[t] = time_step(to_f32(dr[t]) + bias, a.softplus);
      x[t] = dt[t] * uv[t];
      zv[t] = OUT && a.z ? to_f32(zr[t]) : 0.f;
    }
    if (OUT || !(l & 4)) *(f32x4*)&sBC[w][l >> 3][(l >> 2) & 1][4 * (l & 3)] = (f32x4){bc[0], bc[1], bc[2], bc[3]};
    wave_lds_fence();
    if (tb + kScanTok < t1) fetch(tb + kScanTok);
#pragma unroll
    for (int t = 0; t < kScanTok; ++t) {
      if (t >= nt) break;
      const int tok = tb + t;
      if (tok == cur.s) {
        start_state(a, ln, cur.n, h);
        cut = 1;
      }
      const f32x4 Bv = *(const f32x4*)&sBC[w][t][0][4 * ln.j];
      f32x4 Cv;
      if (OUT) Cv = *(const f32x4*)&sBC[w][t][1][4 * ln.j];
      const float dk[4] = {of_channel<0>(dt[t]), of_channel<1>(dt[t]), of_channel<2>(dt[t]), of_channel<3>(dt[t])};
      const float xk[4] = {of_channel<0>(x[t]), of_channel<1>(x[t]), of_channel<2>(x[t]), of_channel<3>(x[t])};
      float s[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[k] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[k][i] = fmaf(fast_exp2(dk[k] * A2[k][i]), h[k][i], xk[k] * Bv[i]);
          if (OUT) s[k] = fmaf(Cv[i], h[k][i], s[k]);
        }
      }
      if (OUT) {
        float yv = quad_total4(s[0], s[1], s[2], s[3], ln.odd, ln.high);
        if constexpr (NW == 1) {
          yv = fmaf(Dc, uv[t], yv);
          if (a.z) yv *= zv[t] * sigmoid_full(zv[t]);
          if (ln.on) py[(int64_t)tok * a.D_] = from_f32<T>(yv);
        } else {
          sY[turn][w][t][l] = yv;
        }
      } else {
        dt_sum += dt[t];
      }
      if (tok + 1 == cur.e) {
        if (OUT && a.final_) ln.store(a, a.final_ + (int64_t)cur.n * a.D_ * a.N, h);
        if (a.cu) {
          int n = cur.n + 1;
          for (; n < a.seqs && a.cu[n + 1] <= tok + 1; ++n)   // sequences without a token
            if (OUT && a.final_) {
              float e[4][4];
              start_state(a, ln, n, e);
              ln.store(a, a.final_ + (int64_t)n * a.D_ * a.N, e);
            }
          if (n < a.seqs) cur = {n, tok + 1, a.cu[n + 1]};
        }
      }
    }
    if constexpr (NW > 1 && OUT) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < kScanTok; ++t) {
        if (t % NW != w || t >= nt) continue;
        float yv = Dc * uv[t];
#pragma unroll
        for (int k = 0; k < NW; ++k) yv += sY[turn][k][t][l];
        if (a.z) yv *= zv[t] * sigmoid_full(zv[t]);
        if (ln.on) py[(int64_t)(tb + t) * a.D_] = from_f32<T>(yv);
      }
      turn ^= 1;
    }
    wave_lds_fence();
  }
  if (!OUT) {
    const int64_t slot = (int64_t)row * a.segs + blockIdx.y;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 v = {h[k][0], h[k][1], h[k][2], h[k][3]};
      ((f32x4*)a.seg_h)[packed_at(slot, a, ln.tile, NW, w, k)] = v;
    }
    if (w == 0) a.seg_dt[(slot * a.tiles + ln.tile) * 64 + l] = dt_sum;
    if (ln.tile == 0 && threadIdx.x == 0) a.seg_cut[slot] = cut;
  }
}

// What comes back over a segment from its end with nothing coming in: a thread-for-thread copy of the backward's carry,
// g <- a (g + C Y) from the last token to the first.
template <typename T, int NW>
__global__ __launch_bounds__(64 * NW) void scan_back_segment_kernel(ScanArgs a) {
  __shared__ float sC[NW][kScanTok][16];
  const Lane<T> ln(a);
  const int l = threadIdx.x & 63, w = ln.w, row = ln.row;
  const int t0 = blockIdx.y * a.seg, t1 = min(a.T, t0 + a.seg);
  const float bias = a.bias ? a.bias[ln.own] : 0.f;
  float A2[4][4], g[4][4], dt_sum = 0.f;
  ln.load(a, a.A, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) { A2[k][i] *= kLog2e; g[k][i] = 0.f; }
  ScanSeq cur = seq_at(a, row, t1 - 1);
  int cut = 0;
  const T* pd = (const T*)a.delta + row * a.db + ln.own;
  const T* pz = a.z ? (const T*)a.z + row * a.zb + ln.own : nullptr;
  const T* pg = (const T*)a.dy + (int64_t)row * a.T * a.D_ + ln.own;
  T dr[kScanTok], zr[kScanTok], gr[kScanTok];
  float bc[4];
  auto fetch = [&](int tb) {
#pragma unroll
    for (int t = 0; t < kScanTok; ++t) {
      const int64_t at = min(tb + t, t1 - 1);
      dr[t] = pd[at * a.dt];
      gr[t] = pg[at * a.D_];
      if (a.z) zr[t] = pz[at * a.zt];
    }
    if (!(l & 32)) ln.fetch_bc(a, a.Cm, row * a.Cb + (int64_t)min(tb + (l >> 2), t1 - 1) * a.Ct, 16 * w + 4 * (l & 3), bc);
  };
  const int last = t0 + (t1 - 1 - t0) / kScanTok * kScanTok;
  fetch(last);
  for (int tb = last; tb >= t0; tb -= kScanTok) {
    const int nt = min(kScanTok, t1 - tb);
    float dt[kScanTok], Y[kScanTok];
#pragma unroll
    for (int t = 0; t < kScanTok; ++t) {
      dt[t] = time_step(to_f32(dr[t]) + bias, a.softplus);
      Y[t] = to_f32(gr[t]);
      if (a.z) {
        const float z = to_f32(zr[t]);
        Y[t] *= z * sigmoid_full(z);
      }
    }
    if (!(l & 32)) *(f32x4*)&sC[w][l >> 2][4 * (l & 3)] = (f32x4){bc[0], bc[1], bc[2], bc[3]};
    wave_lds_fence();
    if (tb > t0) fetch(tb - kScanTok);
#pragma unroll
    for (int t = kScanTok - 1; t >= 0; --t) {
      if (t >= nt) continue;
      const int tok = tb + t;
      if (tok + 1 == cur.e) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) g[k][i] = 0.f;
        if (a.d_final) ln.load(a, a.d_final + (int64_t)cur.n * a.D_ * a.N, g);
      }
      const f32x4 Cv = *(const f32x4*)&sC[w][t][4 * ln.j];
      const float dk[4] = {of_channel<0>(dt[t]), of_channel<1>(dt[t]), of_channel<2>(dt[t]), of_channel<3>(dt[t])};
      const float Yk[4] = {of_channel<0>(Y[t]), of_channel<1>(Y[t]), of_channel<2>(Y[t]), of_channel<3>(Y[t])};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) g[k][i] = fast_exp2(dk[k] * A2[k][i]) * fmaf(Cv[i], Yk[k], g[k][i]);
      dt_sum += dt[t];
      if (tok == cur.s) {
        cut = 1;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) g[k][i] = 0.f;
        if (tok > t0) cur = seq_at(a, row, tok - 1);
      }
    }
    wave_lds_fence();
  }
  const int64_t slot = (int64_t)row * a.segs + blockIdx.y;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const f32x4 v = {g[k][0], g[k][1], g[k][2], g[k][3]};
    ((f32x4*)a.seg_h)[packed_at(slot, a, ln.tile, NW, w, k)] = v;
  }
  if (w == 0) a.seg_dt[(slot * a.tiles + ln.tile) * 64 + l] = dt_sum;
  if (ln.tile == 0 && threadIdx.x == 0) a.seg_cut[slot] = cut;
}

// From what each segment gives by itself to what each segment starts with (BACK: ends with), in place.  Thread = one float4.
template <int NW, bool BACK>
__global__ __launch_bounds__(256) void scan_join_kernel(ScanArgs a) {
  const int l = threadIdx.x & 63, k = threadIdx.x >> 6, w = blockIdx.y, tile = blockIdx.x, row = blockIdx.z;
  const int group = tile / a.tiles_g, base = group * a.per_group + (tile - group * a.tiles_g) * 64;
  const int chan = min(base + 16 * k + (l >> 2), (group + 1) * a.per_group - 1), n0 = 16 * w + 4 * (l & 3);
  float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) A2[i] = n0 + i < a.N ? a.A[(int64_t)chan * a.N + n0 + i] * kLog2e : 0.f;
  f32x4* H = (f32x4*)a.seg_h;
  constexpr int kAhead = 8;
  for (int b = 0; b < a.segs; b += kAhead) {
    f32x4 v[kAhead];
    float d[kAhead];
    int c[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      const int s = min(b + x, a.segs - 1);
      const int64_t slot = (int64_t)row * a.segs + (BACK ? a.segs - 1 - s : s);
      v[x] = H[packed_at(slot, a, tile, NW, w, k)];
      d[x] = a.seg_dt[(slot * a.tiles + tile) * 64 + (l & ~3) + k];
      c[x] = a.seg_cut[slot];
    }
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      if (b + x >= a.segs) break;
      const int64_t slot = (int64_t)row * a.segs + (BACK ? a.segs - 1 - (b + x) : b + x);
      H[packed_at(slot, a, tile, NW, w, k)] = (f32x4){h[0], h[1], h[2], h[3]};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (a state of zero stays zero whatever the decay over the segment has overflowed to)
        const float through = c[x] || h[i] == 0.f ? 0.f : fast_exp2(A2[i] * d[x]) * h[i];
        h[i] = through + v[x][i];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward
constexpr int kSub = 4;   // tokens whose decays and states are in registers

template <typename T, int NW>
__global__ __launch_bounds__(64 * NW) void scan_bwd_kernel(ScanArgs a) {
  constexpr int kBlk = PAL_SCAN_BLOCK;
  __shared__ float sBC[NW][kBlk][2][16];
  __shared__ float sDt[NW][kBlk][64];
  __shared__ f32x4 sH[NW][kBlk / kSub - 1][4][64];
  __shared__ float sS[NW > 1 ? 2 : 1][NW > 1 ? NW : 1][kSub][3][64];
  const Lane<T> ln(a);
  const int l = threadIdx.x & 63, w = ln.w, row = ln.row;
  const int t0 = blockIdx.y * a.seg, t1 = min(a.T, t0 + a.seg);
  const float bias = a.bias ? a.bias[ln.own] : 0.f, Dc = a.D ? a.D[ln.own] : 0.f;
  float A2[4][4], carry[4][4], dA[4][4];
  float dD = 0.f, dbias = 0.f;
  ln.load(a, a.A, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) { A2[k][i] *= kLog2e; carry[k][i] = dA[k][i] = 0.f; }
  const int64_t slot = (int64_t)row * a.segs + blockIdx.y;
  if (t1 < a.T)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 v = ((const f32x4*)a.seg_h)[packed_at(slot, a, ln.tile, NW, w, k)];
#pragma unroll
      for (int i = 0; i < 4; ++i) carry[k][i] = v[i];
    }
  ScanSeq cur = seq_at(a, row, t1 - 1);
  if (t1 == a.T && a.d_init && a.cu)
    for (int n = cur.n + 1; n < a.seqs; ++n) {   // sequences without a token behind the last one
      float e[4][4] = {};
      if (a.d_final) ln.load(a, a.d_final + (int64_t)n * a.D_ * a.N, e);
      ln.store(a, a.d_init + (int64_t)n * a.D_ * a.N, e);
    }
  const T* pu = (const T*)a.u + row * a.ub + ln.own;
  const T* pd = (const T*)a.delta + row * a.db + ln.own;
  const T* pz = a.z ? (const T*)a.z + row * a.zb + ln.own : nullptr;
  const int64_t out0 = (int64_t)row * a.T * a.D_ + ln.own;
  const T* pg = (const T*)a.dy + out0;
  int turn = 0;

  for (int tb = t0 + (t1 - 1 - t0) / kBlk * kBlk; tb >= t0; tb -= kBlk) {
    const int nt = min(kBlk, t1 - tb);
    // ---- the block's time steps, B and C, and its states before tokens 4, 8 and 12
    T ur[kBlk], dr[kBlk];
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const int64_t at = min(tb + t, t1 - 1);
      dr[t] = pd[at * a.dt];
      if (t < kBlk - kSub) ur[t] = pu[at * a.ut];
    }
    {
      const int64_t at = min(tb + (l >> 2), t1 - 1);
      float b[4], c[4];
      ln.fetch_bc(a, a.Bm, row * a.Bb + at * a.Bt, 16 * w + 4 * (l & 3), b);
      ln.fetch_bc(a, a.Cm, row * a.Cb + at * a.Ct, 16 * w + 4 * (l & 3), c);
      *(f32x4*)&sBC[w][l >> 2][0][4 * (l & 3)] = (f32x4){b[0], b[1], b[2], b[3]};
      *(f32x4*)&sBC[w][l >> 2][1][4 * (l & 3)] = (f32x4){c[0], c[1], c[2], c[3]};
    }
    const f32x4* kept = (const f32x4*)a.ckpt + packed_at((int64_t)row * a.ckpts + tb / kBlk, a, ln.tile, NW, w, 0);
    ScanSeq fw = cur.s <= tb ? cur : seq_at(a, row, tb);   // sequence of the block's first token
    const ScanSeq fw0 = fw;
    {
      float h[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 v = kept[k * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[k][i] = v[i];
      }
      wave_lds_fence();
#pragma unroll
      for (int t = 0; t < kBlk; ++t) {
        const float dt = time_step(to_f32(dr[t]) + bias, a.softplus);
        sDt[w][t][l] = dt;
        if (t >= kBlk - kSub || t >= nt) continue;
        const int tok = tb + t;
        if (tok == fw.s) start_state(a, ln, fw.n, h);
        const float x = dt * to_f32(ur[t]);
        const f32x4 Bv = *(const f32x4*)&sBC[w][t][0][4 * ln.j];
        const float dk[4] = {of_channel<0>(dt), of_channel<1>(dt), of_channel<2>(dt), of_channel<3>(dt)};
        const float xk[4] = {of_channel<0>(x), of_channel<1>(x), of_channel<2>(x), of_channel<3>(x)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) h[k][i] = fmaf(fast_exp2(dk[k] * A2[k][i]), h[k][i], xk[k] * Bv[i]);
        if (t % kSub == kSub - 1)
#pragma unroll
          for (int k = 0; k < 4; ++k) sH[w][t / kSub][k][l] = (f32x4){h[k][0], h[k][1], h[k][2], h[k][3]};
        if (tok + 1 == fw.e) fw = seq_at(a, row, min(tok + 1, a.T - 1));
      }
    }
    wave_lds_fence();
    // ---- four tokens at a time from the end
    for (int sub = (nt - 1) / kSub; sub >= 0; --sub) {
      const int ts = tb + sub * kSub, ns = min(kSub, t1 - ts);
      float h[4][4], av[kSub][4][4], ah[kSub][4][4];
      float uv[kSub], zv[kSub], gv[kSub], raw[kSub];
#pragma unroll
      for (int t = 0; t < kSub; ++t) {
        const int64_t at = min(ts + t, t1 - 1);
        uv[t] = to_f32(pu[at * a.ut]);
        raw[t] = to_f32(pd[at * a.dt]) + bias;
        zv[t] = a.z ? to_f32(pz[at * a.zt]) : 0.f;
        gv[t] = ln.on ? to_f32(pg[at * a.D_]) : 0.f;     // (a lane beyond the group adds nothing to dB and dC)
        if (!ln.on) uv[t] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 v = sub ? sH[w][sub ? sub - 1 : 0][k][l] : kept[k * 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[k][i] = v[i];
      }
      ScanSeq sq = cur.s <= ts ? cur : fw0.e > ts ? fw0 : seq_at(a, row, ts);
#pragma unroll
      for (int t = 0; t < kSub; ++t) {
        if (t >= ns) break;
        const int tok = ts + t;
        if (tok == sq.s) start_state(a, ln, sq.n, h);
        const float dt = sDt[w][sub * kSub + t][l], x = dt * uv[t];
        const f32x4 Bv = *(const f32x4*)&sBC[w][sub * kSub + t][0][4 * ln.j];
        const float dk[4] = {of_channel<0>(dt), of_channel<1>(dt), of_channel<2>(dt), of_channel<3>(dt)};
        const float xk[4] = {of_channel<0>(x), of_channel<1>(x), of_channel<2>(x), of_channel<3>(x)};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            av[t][k][i] = fast_exp2(dk[k] * A2[k][i]);
            ah[t][k][i] = av[t][k][i] * h[k][i];
            h[k][i] = fmaf(xk[k], Bv[i], ah[t][k][i]);
          }
        if (tok + 1 == sq.e && t + 1 < ns) sq = seq_at(a, row, tok + 1);
      }
#pragma unroll
      for (int t = kSub - 1; t >= 0; --t) {
        if (t >= ns) continue;
        const int tok = ts + t;
        if (tok + 1 == cur.e) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) carry[k][i] = 0.f;
          if (a.d_final) ln.load(a, a.d_final + (int64_t)cur.n * a.D_ * a.N, carry);
        }
        const float dt = sDt[w][sub * kSub + t][l], x = dt * uv[t];
        const float sz = a.z ? sigmoid_full(zv[t]) : 0.f;
        const float Y = a.z ? gv[t] * zv[t] * sz : gv[t];
        const f32x4 Bv = *(const f32x4*)&sBC[w][sub * kSub + t][0][4 * ln.j];
        const f32x4 Cv = *(const f32x4*)&sBC[w][sub * kSub + t][1][4 * ln.j];
        const float dk[4] = {of_channel<0>(dt), of_channel<1>(dt), of_channel<2>(dt), of_channel<3>(dt)};
        const float xk[4] = {of_channel<0>(x), of_channel<1>(x), of_channel<2>(x), of_channel<3>(x)};
        const float Yk[4] = {of_channel<0>(Y), of_channel<1>(Y), of_channel<2>(Y), of_channel<3>(Y)};
        float gB[4] = {0.f, 0.f, 0.f, 0.f}, gC[4] = {0.f, 0.f, 0.f, 0.f}, sy[4], sb[4], sa[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sy[k] = sb[k] = sa[k] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float hv = fmaf(xk[k], Bv[i], ah[t][k][i]);
            const float g = fmaf(Cv[i], Yk[k], carry[k][i]), p = g * ah[t][k][i];
            gC[i] = fmaf(Yk[k], hv, gC[i]);
            gB[i] = fmaf(g, xk[k], gB[i]);
            sy[k] = fmaf(Cv[i], hv, sy[k]);
            sb[k] = fmaf(g, Bv[i], sb[k]);
            sa[k] = fmaf(p, A2[k][i], sa[k]);
            dA[k][i] = fmaf(p, dk[k], dA[k][i]);
            carry[k][i] = g * av[t][k][i];
          }
        }
        // dB, dC: eight sums over the sixteen quads; lane bits 3, 2, 4 choose among them, bit 5 holds the same twice
        {
          const float p0 = pair_bit3(gB[0], gB[1]), p1 = pair_bit3(gB[2], gB[3]);
          const float p2 = pair_bit3(gC[0], gC[1]), p3 = pair_bit3(gC[2], gC[3]);
          float r0 = pair_bit2(p0, p1), r1 = pair_bit2(p2, p3);
          swap_rows(r0, r1);
          float r = r0 + r1, r2 = r;
          swap_halves(r, r2);
          r += r2;
          if (!(l & 32)) {
            const int which = (l >> 4) & 1, n = 4 * ln.j + ((l >> 2) & 1) * 2 + ((l >> 3) & 1);
            a.part_bc[((((int64_t)row * a.T + tok) * a.tiles + ln.tile) * NW + w) * 32 + which * 16 + n] = r;
          }
        }
        float ty = quad_total4(sy[0], sy[1], sy[2], sy[3], ln.odd, ln.high);
        float tB = quad_total4(sb[0], sb[1], sb[2], sb[3], ln.odd, ln.high);
        float tA = quad_total4(sa[0], sa[1], sa[2], sa[3], ln.odd, ln.high);
        auto finish = [&](float ypre, float sumB, float sumA) {
          ypre = fmaf(Dc, uv[t], ypre);
          dD = fmaf(Y, uv[t], dD);
          const float ddt = fmaf(uv[t], sumB, sumA * 0.6931471806f);
          const float dd = a.softplus && raw[t] <= 20.f ? ddt * sigmoid_full(raw[t]) : ddt;
          if (ln.on) {
            dbias += dd;
            const int64_t at = out0 + (int64_t)tok * a.D_;
            ((T*)a.du)[at] = from_f32<T>(fmaf(dt, sumB, Dc * Y));
            ((T*)a.ddelta)[at] = from_f32<T>(dd);
            if (a.z) ((T*)a.dz)[at] = from_f32<T>(gv[t] * ypre * (sz + zv[t] * sz * (1.f - sz)));
          }
        };
        if constexpr (NW == 1) {
          finish(ty, tB, tA);
        } else {
          sS[turn][w][t][0][l] = ty;
          sS[turn][w][t][1][l] = tB;
          sS[turn][w][t][2][l] = tA;
        }
        if (tok == cur.s) {
          if (a.d_init) ln.store(a, a.d_init + (int64_t)cur.n * a.D_ * a.N, carry);
          if (a.cu) {
            int n = cur.n - 1;
            for (; n >= 0 && a.cu[n] >= tok; --n)   // sequences without a token
              if (a.d_init) {
                float e[4][4] = {};
                if (a.d_final) ln.load(a, a.d_final + (int64_t)n * a.D_ * a.N, e);
                ln.store(a, a.d_init + (int64_t)n * a.D_ * a.N, e);
              }
            if (n >= 0) cur = {n, a.cu[n], tok};
          }
        }
      }
      if constexpr (NW > 1) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
          if (t % NW != w || t >= ns) continue;
          float s3[3];
#pragma unroll
          for (int x = 0; x < 3; ++x) {
            s3[x] = 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) s3[x] += sS[turn][k][t][x][l];
          }
          const int tok = ts + t;
          const float dt = sDt[w][sub * kSub + t][l];
          const float sz = a.z ? sigmoid_full(zv[t]) : 0.f, Y = a.z ? gv[t] * zv[t] * sz : gv[t];
          const float ypre = fmaf(Dc, uv[t], s3[0]);
          dD = fmaf(Y, uv[t], dD);
          const float ddt = fmaf(uv[t], s3[1], s3[2] * 0.6931471806f);
          const float dd = a.softplus && raw[t] <= 20.f ? ddt * sigmoid_full(raw[t]) : ddt;
          if (ln.on) {
            dbias += dd;
            const int64_t at = out0 + (int64_t)tok * a.D_;
            ((T*)a.du)[at] = from_f32<T>(fmaf(dt, s3[1], Dc * Y));
            ((T*)a.ddelta)[at] = from_f32<T>(dd);
            if (a.z) ((T*)a.dz)[at] = from_f32<T>(gv[t] * ypre * (sz + zv[t] * sz * (1.f - sz)));
          }
        }
        turn ^= 1;
      }
    }
    wave_lds_fence();
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    ((f32x4*)a.part_a)[packed_at(slot, a, ln.tile, NW, w, k)] = (f32x4){dA[k][0], dA[k][1], dA[k][2], dA[k][3]};
  float* pc = a.part_c + (((slot * a.tiles + ln.tile) * NW + w) * 64 + l) * 2;
  pc[0] = dD;
  pc[1] = dbias;
}

// dB, dC [rows, T, G, N]: the tiles of a group in their order
template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_rows_kernel(ScanArgs a, int nw) {
  const int64_t per = 2 * (int64_t)a.G * a.N, total = (int64_t)a.rows * a.T * per;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < total; x += (int64_t)gridDim.x * 256) {
    const int64_t tok = x / per;
    const int r = (int)(x - tok * per), which = r >= a.G * a.N, gn = r - which * a.G * a.N, g = gn / a.N, n = gn - g * a.N;
    const float* p = a.part_bc + ((tok * a.tiles + (int64_t)g * a.tiles_g) * nw + (n >> 4)) * 32 + which * 16 + (n & 15);
    float s = 0.f;
    for (int i = 0; i < a.tiles_g; ++i) s += p[(int64_t)i * nw * 32];
    ((T*)(which ? a.dC : a.dB))[tok * a.G * a.N + gn] = from_f32<T>(s);
  }
}

// dA, dD, ddelta_bias: the segments of all rows in their order, in 64 bits.  grid (tiles, waves of a tile, 5): z < 4 the channels
// 16 z .. of dA, z = 4 dD and ddelta_bias; four waves take a quarter of the segments each.
__global__ __launch_bounds__(256) void scan_bwd_params_kernel(ScanArgs a, int nw) {
  __shared__ double s[4][64][4];
  const int l = threadIdx.x & 63, v = threadIdx.x >> 6, tile = blockIdx.x, w = blockIdx.y, z = blockIdx.z;
  const int64_t slots = (int64_t)a.rows * a.segs;
  const int group = tile / a.tiles_g, base = group * a.per_group + (tile - group * a.tiles_g) * 64, end = (group + 1) * a.per_group;
  double t[4] = {0., 0., 0., 0.};
  if (z < 4) {
    for (int64_t i = v; i < slots; i += 4) {
      const f32x4 x = ((const f32x4*)a.part_a)[packed_at(i, a, tile, nw, w, z)];
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] += x[e];
    }
  } else if (w == 0) {
    for (int64_t i = v; i < slots; i += 4)
      for (int k = 0; k < nw; ++k) {
        const float* p = a.part_c + (((i * a.tiles + tile) * nw + k) * 64 + l) * 2;
        t[0] += p[0];
        t[1] += p[1];
      }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s[v][l][e] = t[e];
  __syncthreads();
  if (v) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = s[0][l][e] + s[1][l][e] + s[2][l][e] + s[3][l][e];
  const int q = l >> 2, j = l & 3;
  if (z < 4) {
    const int c = base + 16 * z + q, n0 = 16 * w + 4 * j;
    if (c < end)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n0 + e < a.N) a.dA[(int64_t)c * a.N + n0 + e] = (float)t[e];
  } else if (w == 0) {
    const int c = base + 16 * j + q;
    if (c < end) {
      if (a.dD) a.dD[c] = (float)t[0];
      if (a.dbias) a.dbias[c] = (float)t[1];
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
static int check_scan(const PalScanDims* d) {
  if (!d) return PAL_E_NULL;
  if (d->batch <= 0 || d->seq_len <= 0 || d->n_seqs <= 0 || d->channels <= 0 || d->groups <= 0) return PAL_E_DIM;
  if (d->batch > 65535 || d->channels > 1 << 20 || d->channels % d->groups) return PAL_E_DIM;
  if ((int64_t)d->batch * d->seq_len > (int64_t)1 << 30) return PAL_E_DIM;
  if (d->state < 1 || d->state > PAL_SCAN_MAX_STATE) return PAL_E_DIM;
  if (d->dtype != PAL_DTYPE_F32 && d->dtype != PAL_DTYPE_BF16) return PAL_E_DTYPE;
  if (d->flags & PAL_FLAG_VARLEN) {
    if (d->batch != 1) return PAL_E_VARLEN_BATCH;
  } else if (d->n_seqs != d->batch) {
    return PAL_E_DIM;
  }
  const int64_t strides[] = {d->u_batch, d->delta_batch, d->z_batch, d->B_batch, d->C_batch,
                             d->u_token, d->delta_token, d->z_token, d->B_token, d->C_token};
  for (int64_t s : strides)
    if (s < 0) return PAL_E_DIM;
  return PAL_OK;
}
static int check_scan_tensors(const PalScanDims* d, const PalScanTensors* t) {
  if (!t || !t->u || !t->delta || !t->A || !t->B || !t->C) return PAL_E_NULL;
  if (((d->flags & PAL_FLAG_VARLEN) != 0) != (t->cu_seqlens != nullptr)) return PAL_E_CU_SEQLENS;
  if (((d->flags & PAL_FLAG_HAS_INIT) != 0) != (t->init != nullptr)) return PAL_E_STATE;
  const void* ptrs[] = {t->A, t->init, t->final_, t->checkpoints};
  for (const void* p : ptrs)
    if (p && !is_aligned16(p)) return PAL_E_ALIGN;
  return PAL_OK;
}
static int scan_waves(const PalScanDims* d) { return (d->state + 15) / 16; }
static int64_t scan_tiles(const PalScanDims* d) { return (int64_t)d->groups * ((d->channels / d->groups + 63) / 64); }

// Tokens per segment: enough segments for two waves on every SIMD, at least 64 tokens each
static int scan_segment(const PalScanDims* d) {
  const int64_t waves = scan_tiles(d) * scan_waves(d) * d->batch;
  int64_t segs = (2048 + waves - 1) / waves;
  int64_t seg = (d->seq_len + segs - 1) / segs;
  seg = (seg + PAL_SCAN_BLOCK - 1) / PAL_SCAN_BLOCK * PAL_SCAN_BLOCK;
  if (seg < 64) seg = 64;
  return (int)(seg < d->seq_len ? seg : (d->seq_len + PAL_SCAN_BLOCK - 1) / PAL_SCAN_BLOCK * PAL_SCAN_BLOCK);
}
static void scan_args(ScanArgs& a, const PalScanDims* d, const PalScanTensors* t) {
  a.rows = d->batch; a.T = d->seq_len; a.seqs = d->n_seqs; a.D_ = d->channels; a.N = d->state; a.G = d->groups;
  a.per_group = d->channels / d->groups;
  a.tiles_g = (a.per_group + 63) / 64;
  a.tiles = a.G * a.tiles_g;
  a.softplus = d->softplus;
  a.vec = d->state % 4 == 0;
  a.ub = d->u_batch; a.ut = d->u_token; a.db = d->delta_batch; a.dt = d->delta_token; a.zb = d->z_batch; a.zt = d->z_token;
  a.Bb = d->B_batch; a.Bt = d->B_token; a.Cb = d->C_batch; a.Ct = d->C_token;
  a.seg = scan_segment(d);
  a.segs = (a.T + a.seg - 1) / a.seg;
  a.ckpts = (a.T + PAL_SCAN_BLOCK - 1) / PAL_SCAN_BLOCK;
  if (!t) return;
  a.u = t->u; a.delta = t->delta; a.z = t->z; a.Bm = t->B; a.Cm = t->C;
  a.A = t->A; a.D = t->D; a.bias = t->delta_bias; a.init = t->init;
  a.y = t->y; a.final_ = t->final_; a.ckpt = t->checkpoints; a.cu = t->cu_seqlens;
}
static size_t up256b(size_t x) { return (x + 255) / 256 * 256; }
static size_t packed_bytes(const ScanArgs& a, int nw, int64_t slots) { return up256b((size_t)slots * a.tiles * nw * 4096); }
// segments' states, sums of dt, cuts
static size_t seg_bytes(const ScanArgs& a, int nw) {
  const int64_t slots = (int64_t)a.rows * a.segs;
  return packed_bytes(a, nw, slots) + up256b((size_t)slots * a.tiles * 256) + up256b((size_t)slots * 4);
}
static char* place_segments(ScanArgs& a, int nw, char* p) {
  const int64_t slots = (int64_t)a.rows * a.segs;
  a.seg_h = (float*)p;
  p += packed_bytes(a, nw, slots);
  a.seg_dt = (float*)p;
  p += up256b((size_t)slots * a.tiles * 256);
  a.seg_cut = (int32_t*)p;
  return p + up256b((size_t)slots * 4);
}

template <typename T, int NW>
static int scan_fwd_run(const ScanArgs& a, hipStream_t s) {
  const dim3 grid(a.tiles, a.segs, a.rows);
  if (a.segs > 1) {
    PAL_TIMED_LAUNCH(kKernScanSegment, s, (scan_fwd_kernel<T, NW, false>), grid, dim3(64 * NW), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
    PAL_TIMED_LAUNCH(kKernScanJoin, s, (scan_join_kernel<NW, false>), dim3(a.tiles, NW, a.rows), dim3(256), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
  }
  PAL_TIMED_LAUNCH(kKernScanFwd, s, (scan_fwd_kernel<T, NW, true>), grid, dim3(64 * NW), 0, s, a);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
template <typename T, int NW>
static int scan_bwd_run(const ScanArgs& a, hipStream_t s) {
  const dim3 grid(a.tiles, a.segs, a.rows);
  if (a.segs > 1) {
    PAL_TIMED_LAUNCH(kKernScanSegment, s, (scan_back_segment_kernel<T, NW>), grid, dim3(64 * NW), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
    PAL_TIMED_LAUNCH(kKernScanJoin, s, (scan_join_kernel<NW, true>), dim3(a.tiles, NW, a.rows), dim3(256), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
  }
  PAL_TIMED_LAUNCH(kKernScanBwd, s, (scan_bwd_kernel<T, NW>), grid, dim3(64 * NW), 0, s, a);
  PAL_HIP_LAUNCH_CHECK();
  const int64_t n = 2 * (int64_t)a.rows * a.T * a.G * a.N, blocks = (n + 255) / 256;
  PAL_TIMED_LAUNCH(kKernScanBwdRows, s, scan_bwd_rows_kernel<T>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, a, NW);
  PAL_HIP_LAUNCH_CHECK();
  PAL_TIMED_LAUNCH(kKernScanBwdParams, s, scan_bwd_params_kernel, dim3(a.tiles, NW, 5), dim3(256), 0, s, a, NW);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
template <typename T>
static int scan_fwd_waves(const ScanArgs& a, int nw, hipStream_t s) {
  switch (nw) {
    case 1: return scan_fwd_run<T, 1>(a, s);
    case 2: return scan_fwd_run<T, 2>(a, s);
    case 3: return scan_fwd_run<T, 3>(a, s);
    default: return scan_fwd_run<T, 4>(a, s);
  }
}
template <typename T>
static int scan_bwd_waves(const ScanArgs& a, int nw, hipStream_t s) {
  switch (nw) {
    case 1: return scan_bwd_run<T, 1>(a, s);
    case 2: return scan_bwd_run<T, 2>(a, s);
    case 3: return scan_bwd_run<T, 3>(a, s);
    default: return scan_bwd_run<T, 4>(a, s);
  }
}

}  // namespace pal

extern "C" size_t pal_scan_checkpoint_bytes(const PalScanDims* d) {
  using namespace pal;
  if (check_scan(d) != PAL_OK) return 0;
  ScanArgs a{};
  scan_args(a, d, nullptr);
  return packed_bytes(a, scan_waves(d), (int64_t)a.rows * a.ckpts);
}

extern "C" size_t pal_scan_fwd_workspace_bytes(const PalScanDims* d) {
  using namespace pal;
  if (check_scan(d) != PAL_OK) return 0;
  ScanArgs a{};
  scan_args(a, d, nullptr);
  return a.segs > 1 ? seg_bytes(a, scan_waves(d)) : 0;
}

extern "C" int pal_scan_fwd(const PalScanDims* d, const PalScanTensors* t, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pal;
  if (int rc = check_scan(d)) return rc;
  if (int rc = check_scan_tensors(d, t)) return rc;
  if (!t->y) return PAL_E_NULL;
  if (((d->flags & PAL_FLAG_STORE_FINAL) != 0) != (t->final_ != nullptr)) return PAL_E_STATE;
  ScanArgs a{};
  scan_args(a, d, t);
  const int nw = scan_waves(d);
  if (a.segs > 65535 || a.tiles > (1 << 24)) return PAL_E_DIM;
  if (a.segs > 1) {
    if (!workspace || workspace_bytes < seg_bytes(a, nw)) return PAL_E_WORKSPACE;
    if (!is_aligned16(workspace)) return PAL_E_ALIGN;
    place_segments(a, nw, (char*)workspace);
  }
  hipStream_t s = (hipStream_t)stream;
  return d->dtype == PAL_DTYPE_BF16 ? scan_fwd_waves<bf16_t>(a, nw, s) : scan_fwd_waves<float>(a, nw, s);
}

extern "C" size_t pal_scan_bwd_workspace_bytes(const PalScanDims* d) {
  using namespace pal;
  if (check_scan(d) != PAL_OK) return 0;
  ScanArgs a{};
  scan_args(a, d, nullptr);
  const int nw = scan_waves(d);
  const int64_t slots = (int64_t)a.rows * a.segs;
  return (a.segs > 1 ? seg_bytes(a, nw) : 0) + up256b((size_t)a.rows * a.T * a.tiles * nw * 128) + packed_bytes(a, nw, slots) +
         up256b((size_t)slots * a.tiles * nw * 512);
}

extern "C" int pal_scan_bwd(const PalScanDims* d, const PalScanTensors* t, const PalScanGrads* gr, void* workspace,
                            size_t workspace_bytes, void* stream) {
  using namespace pal;
  if (int rc = check_scan(d)) return rc;
  if (int rc = check_scan_tensors(d, t)) return rc;
  if (!t->checkpoints || !gr || !gr->dy || !gr->du || !gr->ddelta || !gr->dA || !gr->dB || !gr->dC) return PAL_E_NULL;
  if ((t->D != nullptr) != (gr->dD != nullptr) || (t->z != nullptr) != (gr->dz != nullptr) ||
      (t->delta_bias != nullptr) != (gr->ddelta_bias != nullptr))
    return PAL_E_NULL;
  if (gr->d_init && !t->init) return PAL_E_STATE;
  if ((gr->d_init && !is_aligned16(gr->d_init)) || (gr->d_final && !is_aligned16(gr->d_final))) return PAL_E_ALIGN;
  if (!workspace || workspace_bytes < pal_scan_bwd_workspace_bytes(d)) return PAL_E_WORKSPACE;
  if (!is_aligned16(workspace)) return PAL_E_ALIGN;
  ScanArgs a{};
  scan_args(a, d, t);
  const int nw = scan_waves(d);
  if (a.segs > 65535 || a.tiles > (1 << 24)) return PAL_E_DIM;
  a.dy = gr->dy; a.d_final = gr->d_final; a.du = gr->du; a.ddelta = gr->ddelta; a.dA = gr->dA; a.dB = gr->dB; a.dC = gr->dC;
  a.dD = gr->dD; a.dz = gr->dz; a.dbias = gr->ddelta_bias; a.d_init = gr->d_init;
  char* p = (char*)workspace;
  if (a.segs > 1) p = place_segments(a, nw, p);
  a.part_bc = (float*)p;
  p += up256b((size_t)a.rows * a.T * a.tiles * nw * 128);
  a.part_a = (float*)p;
  p += packed_bytes(a, nw, (int64_t)a.rows * a.segs);
  a.part_c = (float*)p;
  hipStream_t s = (hipStream_t)stream;
  return d->dtype == PAL_DTYPE_BF16 ? scan_bwd_waves<bf16_t>(a, nw, s) : scan_bwd_waves<float>(a, nw, s);
}
