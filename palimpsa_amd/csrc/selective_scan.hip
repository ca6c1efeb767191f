// Selective scan: a linear recurrence with a decay of its own for every channel d and state entry n,
//     dt = softplus(delta + bias),   h[d,n] = exp(dt A[d,n]) h[d,n] + dt u[d] B[n],   y[d] = (sum_n C[n] h[d,n] + D u[d]) silu(z[d]).
// Backward, with Y = dy silu(z) and g the gradient of the state after a token (g = C Y + what comes back from the next token):
//     dC[n] = sum_d Y h,  dB[n] = sum_d g dt u,  du = dt sum_n g B + D Y,  ddt = sum_n g (a h') A + u sum_n g B,
//     dA = sum_t dt g (a h'),  dD = sum_t Y u,  dz = dy (sum_n C h + D u) silu'(z),  back to the token before: a g
// with a = exp(dt A), h' the state before the token.  No two entries share a decay, so nothing here is a matrix product.
//
// Bound by the issue of vector instructions: an entry and token take an exponential and four multiplications or fused
// multiply-adds forward (13 + 4 x 2.9 cycles a wave in this mix on this GPU, whatever the order), an exponential and fourteen backward.  A
// wave is 64 channels by 16 state entries.  Forward a lane has one channel and all sixteen: the sum over n stays in the lane, B and C come
// from LDS to all lanes at once.  Backward a lane has 4 channels by 4 entries: sums over d (dB, dC) are then a quarter in registers and the
// rest over sixteen quads, sums over n three quarters in registers and the rest over the four lanes of a quad, and what is done once
// per channel and token (softplus, silu, their derivatives, loads and stores) is one channel for each lane, handed to its quad by lane
// moves.  State sizes above 16 take one wave for each sixteen, which add their sums in LDS.
//
// Where the channels and sequences of a pass are too few waves, the tokens are cut into segments: a first kernel walks each
// segment from zero and leaves its last state and the sum of its dt (the decay over the segment is exp(A sum dt)), a second
// joins them to the states the segments start with, the third is the pass itself.  The backward does the same from the end.  In a packed
// batch segments know nothing of sequences: a token that starts a sequence takes that sequence's initial state in place of the
// state before it, and a segment that holds such a token lets nothing through.
//
// Rows are fetched eight tokens at a time, one block ahead: a lane takes eight neighbouring channels of one token, the block passes
// through LDS, and what a lane computes for its channel goes back the same way.  (A two-byte access per token and array instead
// took eight times the memory instructions.)  Results are stored at the top of the next block, before its fetch: loads and stores
// leave the memory queue in order, and a store issued after a fetch is waited for with it.
//
// For the backward the forward keeps the state before every 8th token in fp32; the backward computes the 8 tokens again, two
// at a time, and keeps a and a h' of two tokens in registers.
//
// Measured (bf16, 1536 channels, N 16, z and D): a call of 1 x 16384 tokens forward 179 us, of 8 x 2048 forward and backward 661 us, of a token of
// 256 sequences 11.7 us.  Under the profiler the first two take 208 and 716: 114 (pass) + 82 (segments) + 11 (join), and 374 (backward) +
// 116 (pass) + 100 + 97 (segments) + 14 (sums) + 9 + 8 (joins).
#include "pal_common.h"
#include "pal_host.h"
#include "pal_profile.h"
#include "rows8.h"
#include "scan_seqs.h"

namespace pal {

struct ScanArgs {
  const void *u, *delta, *z, *Bm, *Cm, *dy;
  const float *A, *D, *bias, *init, *d_final;
  void *y, *du, *ddelta, *dz, *dB, *dC;
  float *final_, *d_init, *ckpt, *dA, *dD, *dbias;
  float *seg_h, *seg_dt, *part_bc, *part_a, *part_c;
  int32_t *seg_cut;
  const int32_t* cu;
  int64_t ub, db, zb, Bb, Cb;                        // strides between batch rows
  int32_t ut, dt, zt, Bt, Ct;                        // and between tokens (below 2^24)
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
// exp2 of x log2(e): for rows in fp32 made up for as above; rows in bf16 are 2^-9 apart, where the rounding of the exponent
// (1.3e-6 of the result at |x| = 20, less below) does not count
template <typename T>
__device__ __forceinline__ float exp_rows(float x) {
  if constexpr (std::is_same<T, float>::value) return exp_full(x);
  else return fast_exp2(x * kLog2e);
}
// log(1 + e) for e >= 0.  The rounding of s = 1 + e is made up for: log(1 + e) - log(s) is (e - (s - 1)) / s to first order.  Below s = 2
// the division changes that by at most 2^-25, half a step of the sum behind it; above, all of it is below 2^-24 and the logarithm
// above 0.69.  So the difference is taken as it is, and held to the 2^-24 that it has below s = 2.
__device__ __forceinline__ float log1p_full(float e) {
  const float s = 1.f + e;
  return fmaf(__builtin_amdgcn_logf(s), 0.6931471806f, __builtin_amdgcn_fmed3f(e - (s - 1.f), -0x1p-24f, 0x1p-24f));
}
// Nothing is moved across by the scheduler.  Independent values go through each kind of operation together: left alone, the scheduler
// walks value by value to save registers, and the product, its exponential and what uses that wait for each other.
__device__ __forceinline__ void stage() { __builtin_amdgcn_sched_barrier(0); }
template <typename T, int K>
__device__ __forceinline__ void exp_rows(const float* x, float* e) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < K; ++i) e[i] = exp_full(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < K; ++i) e[i] = x[i] * kLog2e;
    stage();
#pragma unroll
    for (int i = 0; i < K; ++i) e[i] = fast_exp2(e[i]);
  }
  stage();
}
// K time steps from the raw ones (with their bias); softplus is the identity above 20, as torch computes it (and for a NaN)
template <typename T, int K>
__device__ __forceinline__ void time_steps(const float* raw, float* dt, int softplus) {
  float e[K];
  exp_rows<T, K>(raw, e);
#pragma unroll
  for (int i = 0; i < K; ++i) e[i] = log1p_full(e[i]);
#pragma unroll
  for (int i = 0; i < K; ++i) dt[i] = softplus && raw[i] <= 20.f ? e[i] : raw[i];
}
// K logistic functions
template <typename T, int K>
__device__ __forceinline__ void sigmoids(const float* x, float* sg) {
  float m[K], e[K];
#pragma unroll
  for (int i = 0; i < K; ++i) m[i] = -x[i];
  exp_rows<T, K>(m, e);
#pragma unroll
  for (int i = 0; i < K; ++i) e[i] += 1.f;
  stage();
#pragma unroll
  for (int i = 0; i < K; ++i) sg[i] = fast_rcp(e[i]);
}

// ------------------------------------------------------------------------------------------------ lanes
// lane 4 q + j of a wave: channels 16 k + q (k = 0 .. 3) by entries 4 j + i (i = 0 .. 3) of the state; its own channel is 16 j + q
// (moves inside a quad have a source for every lane: nothing is kept in the target, and the compiler may fold them into their use)
template <int CTRL>
__device__ __forceinline__ float in_quad(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int K>
__device__ __forceinline__ float of_channel(float x) { return in_quad<K * 0x55>(x); }   // the value of the lane that owns channel k
// four sums over a quad: lane j gets the total of p_j
__device__ __forceinline__ float quad_total4(float p0, float p1, float p2, float p3, bool odd, bool high) {
  const float a = (odd ? p1 : p0) + in_quad<0xB1>(odd ? p0 : p1);
  const float b = (odd ? p3 : p2) + in_quad<0xB1>(odd ? p2 : p3);
  return (high ? b : a) + in_quad<0x4E>(high ? a : b);
}

// The lane's number, hidden from the compiler: what rare paths compute from it stays in them instead of being kept in
// registers for all of the loop.
__device__ __forceinline__ int hidden_lane() {
  int l = threadIdx.x & 63;
  asm volatile("" : "+v"(l));
  return l;
}

// A wave's part of a tile of 64 channels: entries 16 w .. of their states.
struct Tile {
  int w, row, tile, group, base, end;      // wave, batch row, tile and its group, first channel of the tile, end of the group
  bool full;                               // all 64 channels of the tile are there
  __device__ __forceinline__ Tile(const ScanArgs& a) {
    w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    tile = blockIdx.x;
    row = blockIdx.z;
    group = tile / a.tiles_g;
    base = group * a.per_group + (tile - group * a.tiles_g) * 64;
    end = (group + 1) * a.per_group;
    full = base + 64 <= end;
  }
};
// Four consecutive entries of a state, zero beyond N.
__device__ __forceinline__ void load4(const ScanArgs& a, const float* s, int n0, float* x) {
  if (a.vec) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n0 < a.N) v = *(const f32x4*)s;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = n0 + i < a.N ? s[i] : 0.f;
  }
}
__device__ __forceinline__ void store4(const ScanArgs& a, float* d, int n0, const float* x) {
  if (a.vec) {
    if (n0 < a.N) *(f32x4*)d = (f32x4){x[0], x[1], x[2], x[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + i < a.N) d[i] = x[i];
  }
}
__device__ __forceinline__ void settle44(float (*x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(x[k][i]));   // (see settle below)
}
// Lanes as columns: lane l has channel l of the tile, x[j][i] entry 4 j + i of the wave's sixteen.
struct Column : Tile {
  unsigned own;                            // own channel; lanes beyond the group have an empty one: rows, states and decays of zero
  bool on;
  __device__ __forceinline__ Column(const ScanArgs& a) : Tile(a) {
    const int c = base + (threadIdx.x & 63);
    on = c < end;
    own = min(c, end - 1);
  }
  // the lane's entries of a [.., channels, N] fp32 array: where sequences start and end, not in the loops over tokens
  __device__ __forceinline__ void load(const ScanArgs& a, const float* p, float (*x)[4]) const {
    const int c = base + hidden_lane();
    const float* s = p + (int64_t)c * a.N + 16 * w;
#pragma unroll
    for (int j = 0; j < 4; ++j) load4(a, s + 4 * j, c < end ? 16 * w + 4 * j : a.N, x[j]);
    settle44(x);
  }
  __device__ __forceinline__ void store(const ScanArgs& a, float* p, const float (*x)[4]) const {
    const int c = base + hidden_lane();
    if (c >= end) return;
    float* d = p + (int64_t)c * a.N + 16 * w;
#pragma unroll
    for (int j = 0; j < 4; ++j) store4(a, d + 4 * j, 16 * w + 4 * j, x[j]);
  }
  __device__ __forceinline__ void clear_beyond(const ScanArgs& a, float (*x)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = 16 * w + 4 * j + i < a.N ? x[j][i] : 0.f;
  }
  static __device__ __forceinline__ unsigned packed(int j) { return 64 * j + (threadIdx.x & 63); }
};
// Lanes as quads: x[k][i] is channel 16 k + q of the tile, entry 4 j + i of the wave's sixteen, for lane 4 q + j.
struct Lane : Tile {
  int j;                                   // place in the quad
  unsigned own;                            // own channel
  bool on, odd, high;
  __device__ __forceinline__ Lane(const ScanArgs& a) : Tile(a) {
    const int l = threadIdx.x & 63;
    j = l & 3;
    odd = j & 1; high = j & 2;
    const int c = base + 16 * j + (l >> 2);
    on = c < end;
    own = min(c, end - 1);
  }
  __device__ __forceinline__ void load(const ScanArgs& a, const float* p, float (*x)[4]) const {
    const int l = hidden_lane(), n0 = 16 * w + 4 * (l & 3);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = base + 16 * k + (l >> 2);
      load4(a, p + (int64_t)c * a.N + n0, c < end ? n0 : a.N, x[k]);
    }
    settle44(x);
  }
  __device__ __forceinline__ void store(const ScanArgs& a, float* p, const float (*x)[4]) const {
    const int l = hidden_lane(), n0 = 16 * w + 4 * (l & 3);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = base + 16 * k + (l >> 2);
      if (c < end) store4(a, p + (int64_t)c * a.N + n0, n0, x[k]);
    }
  }
  __device__ __forceinline__ int entries(const ScanArgs& a) const { return a.N - 16 * w - 4 * (hidden_lane() & 3); }   // of the lane's four
  __device__ __forceinline__ void clear_beyond(const ScanArgs& a, float (*x)[4]) const {
    const int have = entries(a);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[k][i] = i < have ? x[k][i] : 0.f;
  }
  static __device__ __forceinline__ unsigned packed(int k) { return 64 * (threadIdx.x & 3) + 16 * k + ((threadIdx.x & 63) >> 2); }
};
// An element of a row: the row's address is the same for the whole wave, the lane adds 32 bits.  The empty assembly keeps the address
// in scalar registers: left alone, the compiler adds the lane's part first and carries one 64-bit address per array and lane
// through the loops.
#define PAL_GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ PAL_GLOBAL T* row_element(const T* row, unsigned bytes) {
  const uint64_t p = (uint64_t)row;
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)p), hi = __builtin_amdgcn_readfirstlane((int)(p >> 32));
  auto base = (PAL_GLOBAL char*)((uint64_t)hi << 32 | lo);
  asm("" : "+s"(base));
  asm("" : "+v"(bytes));
  return (PAL_GLOBAL T*)(base + bytes);
}
template <typename T>
__device__ __forceinline__ T row_load(const T* row, unsigned i) { return *row_element(row, i * (unsigned)sizeof(T)); }
template <typename T>
__device__ __forceinline__ void row_store(T* row, unsigned i, T x) { *row_element(row, i * (unsigned)sizeof(T)) = x; }
// A load that only some paths make has to be waited for on those paths: where they meet the others again, the compiler would wait for
// every load in flight on any of them, the next block's rows among them.  The empty assembly is a use of the value.
__device__ __forceinline__ void settle(float& x) { asm volatile("" : "+v"(x)); }

// Four entries of B or C, from entry n on (zero beyond N), as fetched.  p: the group's entries of the block's first token; the
// lane's token is `bytes` behind it.
template <typename T>
struct Four {
  typename Raw4<T>::type v;
  __device__ __forceinline__ void fetch(const ScanArgs& a, const T* p, unsigned bytes, int n) {
    typedef typename Raw4<T>::type any __attribute__((aligned(sizeof(T))));
    if (a.vec) {
      v = *(const PAL_GLOBAL any*)row_element(p, bytes + (n < a.N ? n : 0) * (unsigned)sizeof(T));
    } else {
      asm volatile("" : "+v"(n));
      const T* q = (const T*)((const char*)p + bytes) + n;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = n + i < a.N ? q[i] : (T)0.f;
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = (float)v[i];
        settle(x[i]);
        v[i] = (T)x[i];
      }
    }
  }
  __device__ __forceinline__ f32x4 get(const ScanArgs& a, int n) const {
    const f32x4 x = {(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    return n < a.N ? x : (f32x4){0.f, 0.f, 0.f, 0.f};
  }
};
// A wave's entries in scratch: a float4 for entries 4 j .. of every channel of the tile, j first
__device__ __forceinline__ int64_t packed_at(int64_t slot, const ScanArgs& a, int tile, int nw, int w, int j) {
  return (((slot * a.tiles + tile) * nw + w) * 4 + j) * 64;
}
template <typename L>
__device__ __forceinline__ void load_packed(const L&, const float* p, int64_t at, float (*x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const f32x4 v = row_load((const f32x4*)p + at, L::packed(k));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[k][i] = v[i];
  }
}
template <typename L>
__device__ __forceinline__ void store_packed(const L&, float* p, int64_t at, const float (*x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) row_store((f32x4*)p + at, L::packed(k), (f32x4){x[k][0], x[k][1], x[k][2], x[k][3]});
}
__device__ __forceinline__ void zero44(float (*x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[k][i] = 0.f;
}
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// a sequence's entries of a [seqs, channels, N] array, or zero where there is none
template <typename L>
__device__ __forceinline__ void load_state(const ScanArgs& a, const L& ln, const float* p, int seq, float (*h)[4]) {
  if (p) ln.load(a, p + (int64_t)seq * a.D_ * a.N, h);
  else zero44(h);
}
template <typename L>
__device__ __forceinline__ void store_state(const ScanArgs& a, const L& ln, float* p, int seq, const float (*h)[4]) {
  ln.store(a, p + (int64_t)seq * a.D_ * a.N, h);
}
// sequences [n, end) have no token: what they start with is what they end with
template <typename L>
__device__ __forceinline__ void hand_over(const ScanArgs& a, const L& ln, const float* from, float* to, int n, int end) {
  if (!to) return;
  for (; n < end; ++n) {
    float x[4][4];
    load_state(a, ln, from, n, x);
    store_state(a, ln, to, n, x);
  }
}
// the tokens of a block that are walked: all of them, known to the compiler, or [lo, hi)
struct Whole {
  static constexpr bool whole = true;
  int lo, hi;
};
struct Part {
  static constexpr bool whole = false;
  int lo, hi;
};
template <typename R>
__device__ __forceinline__ bool walks(const R& r, int t) { return R::whole || (t >= r.lo && t < r.hi); }

constexpr int kTok = PAL_SCAN_BLOCK;   // tokens of a block

// Entries beyond N have B = C = 0 and no decay, so they stay zero, unless a factor is infinite: inf x 0 is no number, and would get into the
// sums over n.  A block in which one is takes the path that clears them; this looks for it in `most`, the largest of the factors.  (A factor
// that is no number makes every entry of its channel one, until its sequence ends, and need not be looked for.)  In what a segment leaves they
// are whatever they are: it is cleared where it is read.  Passes over states of a multiple of 16 entries are kernels of their own (FULL):
// the second path and the looking take 1 to 3 % of a forward call, and 4 x 2048 tokens of 1536 channels forward and backward from 347 to 364 us
// for N 8, from 695 to 743 for N 24 (bf16; 575 to 503 and 958 to 961 in fp32).
__device__ __forceinline__ bool any_infinite(float most) { return __builtin_amdgcn_ballot_w64(most == INFINITY) != 0; }

// A block of one array: lane l takes channels 8 (l % 8) .. of token l / 8 (of the last token where the block has fewer).  Whole tiles
// without a branch; of the last tile of a group what is there, the channels beyond it are zero.
template <typename T>
struct BlockRows {
  Piece8<T> v;
  // row: the block's first token; left: tokens behind it
  __device__ __forceinline__ void fetch(const Tile& ln, const T* row, int stride, int left) {
    const int l = threadIdx.x & 63;
    const unsigned at = __umul24(min(l >> 3, left), stride) + ln.base + 8 * (l & 7);
    if (ln.full) {
      v.load(row_element(row, at * (unsigned)sizeof(T)));
    } else {
      const int h = hidden_lane();
      load_piece(v, row + __umul24(min(h >> 3, left), stride) + ln.base + 8 * (h & 7), ln.end - ln.base - 8 * (h & 7));
      v.settle();
    }
  }
  __device__ __forceinline__ void to_lds(T (*to)[64]) const {
    const int l = threadIdx.x & 63;
    *(Piece8<T>*)&to[l >> 3][8 * (l & 7)] = v;
  }
  // and back: a block of results, nt tokens of it
  __device__ __forceinline__ void from_lds(const T (*from)[64]) {
    const int l = threadIdx.x & 63;
    v = *(const Piece8<T>*)&from[l >> 3][8 * (l & 7)];
  }
  __device__ __forceinline__ void store(const Tile& ln, T* row, int stride, int nt) const {
    const int l = threadIdx.x & 63;
    const unsigned at = __umul24(l >> 3, stride) + ln.base + 8 * (l & 7);
    if (ln.full && nt == kTok) {
      v.store(row_element(row, at * (unsigned)sizeof(T)));
    } else {
      const int h = hidden_lane();
      T* to = row + __umul24(h >> 3, stride) + ln.base + 8 * (h & 7);
      if ((h >> 3) < nt)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < ln.end - ln.base - 8 * (h & 7)) to[e] = v.at(e);
    }
  }
};
// element of a block in LDS that belongs to a lane's own channel
__device__ __forceinline__ int own_at() { return 16 * (threadIdx.x & 3) + ((threadIdx.x & 63) >> 2); }

// B and C of a block of tokens, fetched a block ahead by the lanes and read from LDS by all at once.  (Read by the scalar unit and
// taken from scalar registers they cost the same: 112 and 110 us of 16384 tokens of 1536 channels, and rows have to be whole and aligned.)
template <typename T, int M>
struct TokenRows {
  const T* p[M];
  int stride[M];
  Four<T> r[M];
  __device__ __forceinline__ void fetch(const ScanArgs& a, int tb, int left, int w) {
    const int l = threadIdx.x & 63, t = min((l >> 2) & 7, left);   // lane l: four entries of token l / 4 (of the last token there is)
#pragma unroll
    for (int m = 0; m < M; ++m) r[m].fetch(a, p[m] + (int64_t)tb * stride[m], __umul24(t, stride[m]) * (unsigned)sizeof(T), 16 * w + 4 * (l & 3));
  }
  __device__ __forceinline__ void to_lds(const ScanArgs& a, float (*s)[M][16], int w) const {
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int m = 0; m < M; ++m) *(f32x4*)&s[(l >> 2) & 7][m][4 * (l & 3)] = r[m].get(a, 16 * w + 4 * (l & 3));   // (the upper half holds the same)
  }
};
// decays of a token: the products, then the exponentials (see stage)
__device__ __forceinline__ void decays(float (*e)[4], float dt, const float (*A2)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) e[j][i] = dt * A2[j][i];
  stage();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) e[j][i] = fast_exp2(e[j][i]);
}

// ------------------------------------------------------------------------------------------------ forward
// OUT: the pass itself.  Otherwise the walk of a segment from zero: its last state, the sum of its dt, and whether a sequence starts in it.
template <typename T, int NW, bool OUT, bool FULL>
__global__ __launch_bounds__(64 * NW, 3) void scan_fwd_kernel(ScanArgs a) {
  constexpr int M = OUT ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float sBC[NW][kTok][M][16];
  __shared__ __attribute__((aligned(16))) T sRow[NW][OUT ? 3 : 2][kTok][64];   // u, delta, z
  __shared__ __attribute__((aligned(16))) T sOut[OUT && NW == 1 ? kTok : 1][64];
  __shared__ float sY[NW > 1 && OUT ? 2 : 1][NW > 1 && OUT ? NW : 1][kTok][64];
  Column ln(a);
  if (NW == 1) ln.w = 0;      // (known to the compiler)
  const int l = threadIdx.x & 63, w = ln.w, row = ln.row;
  const int t0 = blockIdx.y * a.seg, t1 = min(a.T, t0 + a.seg);
  const float bias = a.bias && ln.on ? a.bias[ln.own] : 0.f, Dc = a.D ? a.D[ln.own] : 0.f;
  float A2[4][4], h[4][4], dt_sum = 0.f;
  ln.load(a, a.A, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[k][i] *= kLog2e;
  const bool beyond = OUT && !FULL && 16 * (w + 1) > a.N;      // entries beyond N in this wave
  ScanSeq cur = seq_at(a, row, t0);
  int cut = 0;
  // (of a dense batch in segments the join hands on the initial state too: the last segment may be writing the final state there already)
  const bool joined = OUT && a.segs > 1 && !a.cu;
  if (OUT && (joined || (t0 > 0 && cur.s != t0))) load_packed(ln, a.seg_h, packed_at((int64_t)row * a.segs + blockIdx.y, a, ln.tile, NW, w, 0), h);
  else zero44(h);
  if (beyond) ln.clear_beyond(a, h);
  if (OUT && t0 == 0 && a.cu) hand_over(a, ln, a.init, a.final_, 0, cur.n);   // sequences without a token before the first one
  const T* pu = (const T*)a.u + row * a.ub;
  const T* pd = (const T*)a.delta + row * a.db;
  const T* pz = a.z ? (const T*)a.z + row * a.zb : nullptr;
  T* py = (T*)a.y + (int64_t)row * a.T * a.D_;
  TokenRows<T, M> bc;
  bc.p[0] = (const T*)a.Bm + row * a.Bb + (int64_t)ln.group * a.N;
  bc.stride[0] = a.Bt;
  if constexpr (OUT) {
    bc.p[1] = (const T*)a.Cm + row * a.Cb + (int64_t)ln.group * a.N;
    bc.stride[1] = a.Ct;
  }

  BlockRows<T> ru, rd, rz;
  auto fetch = [&](int tb) {
    const int left = min(kTok, t1 - tb) - 1;
    ru.fetch(ln, pu + (int64_t)tb * a.ut, a.ut, left);
    rd.fetch(ln, pd + (int64_t)tb * a.dt, a.dt, left);
    if (OUT && a.z) rz.fetch(ln, pz + (int64_t)tb * a.zt, a.zt, left);
    bc.fetch(a, tb, left, w);
  };
  fetch(t0);
  int turn = 0;
  for (int tb = t0; tb < t1; tb += kTok) {
    ru.to_lds(sRow[w][0]);
    rd.to_lds(sRow[w][1]);
    if (OUT && a.z) rz.to_lds(sRow[w][OUT ? 2 : 0]);
    bc.to_lds(a, sBC[w], w);
    if constexpr (OUT && NW == 1) {
      if (tb > t0) {
        BlockRows<T> done;
        done.from_lds(sOut);
        done.store(ln, py + (int64_t)(tb - kTok) * a.D_, a.D_, kTok);
      }
    }
    if (OUT && a.ckpt) store_packed(ln, a.ckpt, packed_at((int64_t)row * a.ckpts + tb / kTok, a, ln.tile, NW, w, 0), h);
    wave_lds_fence();
    if (tb + kTok < t1) fetch(tb + kTok);
    const int nt = min(kTok, t1 - tb);
    float dt[kTok], uv[kTok], gate[kTok], raw[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      uv[t] = to_f32(sRow[w][0][t][l]);
      raw[t] = to_f32(sRow[w][1][t][l]) + bias;
      gate[t] = 1.f;
    }
    stage();
    time_steps<T, kTok>(raw, dt, a.softplus);
    if (OUT && a.z) {
#pragma unroll
      for (int t = 0; t < kTok; ++t) raw[t] = to_f32(sRow[w][OUT ? 2 : 0][t][l]);
      stage();
      sigmoids<T, kTok>(raw, gate);
#pragma unroll
      for (int t = 0; t < kTok; ++t) gate[t] *= raw[t];
    }
    bool clear = false;
    if (beyond) {
      float most = 0.f;
#pragma unroll
      for (int t = 0; t < kTok; ++t) most = fmaxf(fmaxf(most, fabsf(dt[t])), fabsf(dt[t] * uv[t]));
      clear = any_infinite(most);
    }
    auto walk = [&](auto r) {
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        if (!walks(r, t)) continue;
        float dtt = dt[t], e[4][4], s[4];
        settle(dtt);          // (the two walks have the same products, which the compiler would else compute before choosing between them)
        const float x = dtt * uv[t];
        const f32x4 *B = (const f32x4*)sBC[w][t][0], *C = (const f32x4*)sBC[w][t][M - 1];
        stage();
        decays(e, dtt, A2);
        stage();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) h[j][i] = fmaf(e[j][i], h[j][i], x * B[j][i]);
        if (beyond && !decltype(r)::whole && clear) ln.clear_beyond(a, h);
        stage();
        if constexpr (OUT) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = j ? fmaf(C[j][i], h[j][i], s[i]) : C[j][i] * h[j][i];
          const float y = (s[0] + s[1]) + (s[2] + s[3]);
          if constexpr (NW == 1) sOut[t][l] = from_f32<T>(fmaf(Dc, uv[t], y) * gate[t]);
          else sY[turn][w][t][l] = y;
        } else {
          dt_sum += dt[t];
        }
      }
    };
    for (int lo = 0, hi; lo < nt; lo = hi) {   // the parts of the block that belong to one sequence each: one, nearly always
      if (tb + lo == cur.s) {
        if (!joined) load_state(a, ln, a.init, cur.n, h);
        cut = 1;
      }
      hi = max(lo + 1, min(clear ? min(nt, kTok - 1) : nt, cur.e - tb));
      if (hi - lo == kTok) walk(Whole{0, 0});
      else walk(Part{lo, hi});
      if (tb + hi == cur.e) {
        if (OUT && a.final_) store_state(a, ln, a.final_, cur.n, h);
        if (a.cu) {
          const ScanSeq next = next_seq(a, cur);
          if (OUT) hand_over(a, ln, a.init, a.final_, cur.n + 1, next.n);
          cur = next;
        }
      }
    }
    if constexpr (NW > 1 && OUT) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        if (t % NW != w || t >= nt) continue;
        float y = Dc * uv[t];
#pragma unroll
        for (int k = 0; k < NW; ++k) y += sY[turn][k][t][l];
        if (ln.on) row_store(py + (int64_t)(tb + t) * a.D_, ln.own, from_f32<T>(y * gate[t]));
      }
      turn ^= 1;
    }
    wave_lds_fence();
  }
  if constexpr (OUT && NW == 1) {
    const int tb = t0 + (t1 - 1 - t0) / kTok * kTok;
    BlockRows<T> done;
    done.from_lds(sOut);
    done.store(ln, py + (int64_t)tb * a.D_, a.D_, t1 - tb);
  }
  if (!OUT) {
    const int64_t slot = (int64_t)row * a.segs + blockIdx.y;
    store_packed(ln, a.seg_h, packed_at(slot, a, ln.tile, NW, w, 0), h);
    if (w == 0) a.seg_dt[(slot * a.tiles + ln.tile) * 64 + l] = dt_sum;
    if (ln.tile == 0 && threadIdx.x == 0) a.seg_cut[slot] = cut;
  }
}

// A few tokens: the state is all the traffic, and a wave of the kernel above would wait for one block of it at a time.  Thread = four
// entries of the state of one channel, in the order of memory; LPC threads a channel add their sums.  256 x 1 tokens of 1536 channels, N 16:
// a call of 11.8 us, 4.5 TB/s (18.1 in the kernel above; at eight tokens the two are equal).  The sum over a channel's threads is by lane moves, which
// takes a power of two of them: N 4, 8, 16, 32 and 64; the others go to the kernel above (N 12, 24, 48: 16, 28, 44 us; N 32, 64 here 20, 35).
constexpr int kStepTokens = 4;
template <int LPC>
__device__ __forceinline__ float channel_sum(float x) {
  if constexpr (LPC > 1) x += in_quad<0xB1>(x);
  if constexpr (LPC > 2) x += in_quad<0x4E>(x);
  if constexpr (LPC > 4) x += in_quad<0x141>(x);   // row_half_mirror
  if constexpr (LPC > 8) x += in_quad<0x140>(x);   // row_mirror
  return x;
}
template <typename T, int LPC>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
  constexpr int N = 4 * LPC;
  const int c = blockIdx.x * (256 / LPC) + threadIdx.x / LPC, j = threadIdx.x % LPC, b = blockIdx.y;
  if (c >= a.D_) return;
  const int64_t at = ((int64_t)b * a.D_ + c) * N + 4 * j;
  f32x4 h = {0.f, 0.f, 0.f, 0.f};
  if (a.init) h = *(const f32x4*)(a.init + at);
  const f32x4 A = *(const f32x4*)(a.A + (int64_t)c * N + 4 * j);
  const float bias = a.bias ? a.bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
  const int64_t bc = (int64_t)(c / a.per_group) * N + 4 * j;
  typedef typename Raw4<T>::type any __attribute__((aligned(sizeof(T))));
  for (int t = 0; t < a.T; ++t) {
    const float u = to_f32(((const T*)a.u)[b * a.ub + (int64_t)t * a.ut + c]);
    const float raw = to_f32(((const T*)a.delta)[b * a.db + (int64_t)t * a.dt + c]) + bias;
    const any Bv = *(const any*)((const T*)a.Bm + b * a.Bb + (int64_t)t * a.Bt + bc);
    const any Cv = *(const any*)((const T*)a.Cm + b * a.Cb + (int64_t)t * a.Ct + bc);
    float gate = 1.f;
    if (a.z) {
      const float z = to_f32(((const T*)a.z)[b * a.zb + (int64_t)t * a.zt + c]);
      sigmoids<T, 1>(&z, &gate);
      gate *= z;
    }
    float dt;
    time_steps<T, 1>(&raw, &dt, a.softplus);
    const float x = dt * u;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = fmaf(fast_exp2(dt * (A[i] * kLog2e)), h[i], x * (float)Bv[i]);
      y = fmaf((float)Cv[i], h[i], y);
    }
    y = channel_sum<LPC>(y);
    if (j == 0) ((T*)a.y)[((int64_t)b * a.T + t) * a.D_ + c] = from_f32<T>(fmaf(Dc, u, y) * gate);
  }
  if (a.final_) *(f32x4*)(a.final_ + at) = h;
}

// What comes back over a segment from its end with nothing coming in: the backward's carry, g <- a (g + C Y) from the last
// token to the first.
template <typename T, int NW>
__global__ __launch_bounds__(64 * NW) void scan_back_segment_kernel(ScanArgs a) {
  __shared__ __attribute__((aligned(16))) float sC[NW][kTok][1][16];
  __shared__ __attribute__((aligned(16))) T sRow[NW][3][kTok][64];   // dy, delta, z
  Column ln(a);
  if (NW == 1) ln.w = 0;      // (known to the compiler)
  const int l = threadIdx.x & 63, w = ln.w, row = ln.row;
  const int t0 = blockIdx.y * a.seg, t1 = min(a.T, t0 + a.seg);
  const float bias = a.bias && ln.on ? a.bias[ln.own] : 0.f;
  float A2[4][4], g[4][4], dt_sum = 0.f;
  ln.load(a, a.A, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[k][i] *= kLog2e;
  zero44(g);
  ScanSeq cur = seq_at(a, row, t1 - 1);
  int cut = 0;
  const T* pd = (const T*)a.delta + row * a.db;
  const T* pz = a.z ? (const T*)a.z + row * a.zb : nullptr;
  const T* pg = (const T*)a.dy + (int64_t)row * a.T * a.D_;
  TokenRows<T, 1> rc;
  rc.p[0] = (const T*)a.Cm + row * a.Cb + (int64_t)ln.group * a.N;
  rc.stride[0] = a.Ct;
  BlockRows<T> rg, rd, rz;
  auto fetch = [&](int tb) {
    const int left = min(kTok, t1 - tb) - 1;
    rg.fetch(ln, pg + (int64_t)tb * a.D_, a.D_, left);
    rd.fetch(ln, pd + (int64_t)tb * a.dt, a.dt, left);
    if (a.z) rz.fetch(ln, pz + (int64_t)tb * a.zt, a.zt, left);
    rc.fetch(a, tb, left, w);
  };
  const int last = t0 + (t1 - 1 - t0) / kTok * kTok;
  fetch(last);
  for (int tb = last; tb >= t0; tb -= kTok) {
    rg.to_lds(sRow[w][0]);
    rd.to_lds(sRow[w][1]);
    if (a.z) rz.to_lds(sRow[w][2]);
    rc.to_lds(a, sC[w], w);
    wave_lds_fence();
    if (tb > t0) fetch(tb - kTok);
    const int nt = min(kTok, t1 - tb);
    float dt[kTok], Y[kTok], raw[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      raw[t] = to_f32(sRow[w][1][t][l]) + bias;
      Y[t] = to_f32(sRow[w][0][t][l]);
    }
    stage();
    time_steps<T, kTok>(raw, dt, a.softplus);
    if (a.z) {
      float sg[kTok];
#pragma unroll
      for (int t = 0; t < kTok; ++t) raw[t] = to_f32(sRow[w][2][t][l]);
      stage();
      sigmoids<T, kTok>(raw, sg);
#pragma unroll
      for (int t = 0; t < kTok; ++t) Y[t] *= raw[t] * sg[t];
    }
    auto walk = [&](auto r) {
#pragma unroll
      for (int t = kTok - 1; t >= 0; --t) {
        if (!walks(r, t)) continue;
        const f32x4* C = (const f32x4*)sC[w][t][0];
        float dtt = dt[t], e[4][4];
        settle(dtt);          // (as in the forward)
        stage();
        decays(e, dtt, A2);
        stage();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) g[j][i] = fmaf(C[j][i], Y[t], g[j][i]);
        stage();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) g[j][i] *= e[j][i];
        dt_sum += dt[t];
      }
    };
    for (int hi = nt, lo; hi > 0; hi = lo) {
      if (tb + hi == cur.e) load_state(a, ln, a.d_final, cur.n, g);
      lo = min(hi - 1, max(0, cur.s - tb));
      if (hi - lo == kTok) walk(Whole{0, 0});
      else walk(Part{lo, hi});
      if (tb + lo == cur.s) {
        cut = 1;
        zero44(g);
        if (a.cu) cur = prev_seq(a, cur);
      }
    }
    wave_lds_fence();
  }
  const int64_t slot = (int64_t)row * a.segs + blockIdx.y;
  store_packed(ln, a.seg_h, packed_at(slot, a, ln.tile, NW, w, 0), g);
  if (w == 0) a.seg_dt[(slot * a.tiles + ln.tile) * 64 + l] = dt_sum;
  if (ln.tile == 0 && threadIdx.x == 0) a.seg_cut[slot] = cut;
}

// From what each segment gives by itself to what each segment starts with (BACK: ends with), in place.  A workgroup has one float4 of
// every channel of a tile (entries 4 j ..); its waves (up to sixteen) take a run of the segments each: what a run gives by itself goes through
// LDS, every wave adds up the runs in front of its own, and walks its run again with what it starts with.  One wave over all of the
// 128 segments of 16384 tokens waited for sixteen batches of loads in turn: 27 us, so split 10.5.
constexpr int kJoinWaves = 16, kJoinAhead = 8;
// INF: a state may be infinite.  The decay of many tokens at once, which may be zero in fp32, then leaves it as it is.
template <bool INF>
__device__ __forceinline__ void join_step(float* h, const float* A2, float d, int cut, const f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (a state of zero stays zero whatever the decay over the segment has overflowed to)
    const float x = A2[i] * d, through = INF && fabsf(h[i]) == INFINITY && x > -INFINITY ? h[i] : fast_exp2(x) * h[i];
    h[i] = (((cut != 0) | (h[i] == 0.f)) ? 0.f : through) + v[i];
  }
}
__device__ __forceinline__ float largest(float m, const float* x) {
  return fmaxf(fmaxf(fmaxf(m, fabsf(x[0])), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}
template <int NW, bool BACK>
__global__ __launch_bounds__(64 * kJoinWaves) void scan_join_kernel(ScanArgs a) {
  __shared__ f32x4 sH[kJoinWaves][64];
  __shared__ float sD[kJoinWaves][64];
  __shared__ int sCut[kJoinWaves], sInf[kJoinWaves];
  const int l = threadIdx.x & 63, v = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = blockIdx.x, w = blockIdx.y >> 2, j = blockIdx.y & 3, row = blockIdx.z;
  const int group = tile / a.tiles_g, base = group * a.per_group + (tile - group * a.tiles_g) * 64;
  const int chan = base + l, n0 = chan < (group + 1) * a.per_group ? 16 * w + 4 * j : a.N;   // (lanes beyond the group: nothing)
  float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f}, d_sum = 0.f;
  load4(a, a.A + (int64_t)chan * a.N + n0, n0, A2);
#pragma unroll
  for (int i = 0; i < 4; ++i) A2[i] *= kLog2e;
  f32x4* H = (f32x4*)a.seg_h;
  const int waves = blockDim.x >> 6, per = (a.segs + waves - 1) / waves, s0 = min(v * per, a.segs), s1 = min(s0 + per, a.segs);
  int any = 0;
  constexpr int kAhead = kJoinAhead;
  f32x4 x[kAhead];
  float d[kAhead];
  int c[kAhead];
  auto slot_of = [&](int s) { return (int64_t)row * a.segs + (BACK ? a.segs - 1 - s : s); };
  auto fetch = [&](int b) {
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const int64_t slot = slot_of(min(b + y, a.segs - 1));
      x[y] = H[packed_at(slot, a, tile, NW, w, j) + l];
      d[y] = a.seg_dt[(slot * a.tiles + tile) * 64 + l];
      c[y] = a.seg_cut[slot];
    }
  };
  // infinite states are looked for once a batch, here and in the state that comes in: looked for in every step they cost 2.7 us of 10.6, so 0.6
  bool inf = false;
  for (int b = s0; b < s1; b += kAhead) {
    fetch(b);
    float most = 0.f;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) most = largest(most, (const float*)&x[y]);
    inf |= any_infinite(most);
    auto walk = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
      for (int y = 0; y < kAhead; ++y) {
        if (b + y >= s1) break;
        join_step<decltype(careful)::value>(h, A2, d[y], c[y], x[y]);
        d_sum += d[y];
        any |= c[y];
      }
    };
    if (inf) walk(std::true_type());
    else walk(std::false_type());
  }
  float first[4] = {0.f, 0.f, 0.f, 0.f};
  if (!BACK && v == 0 && a.init && !a.cu) {   // (the first segment's own state has it already, and lets nothing through)
    load4(a, a.init + ((int64_t)row * a.D_ + chan) * a.N + n0, n0, first);
    inf |= any_infinite(largest(0.f, first));
  }
  sH[v][l] = (f32x4){h[0], h[1], h[2], h[3]};
  sD[v][l] = d_sum;
  if (l == 0) {
    sCut[v] = any;
    sInf[v] = inf;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = first[i];
  auto hand_on = [&](auto careful) __attribute__((always_inline)) {
    constexpr bool INF = decltype(careful)::value;
#pragma unroll 4
    for (int y = 0; y < v; ++y) join_step<INF>(h, A2, sD[y][l], sCut[y], sH[y][l]);
    for (int b = s0; b < s1; b += kAhead) {
      if (per > kAhead) fetch(b);       // (else they are still in registers)
#pragma unroll
      for (int y = 0; y < kAhead; ++y) {
        if (b + y >= s1) break;
        H[packed_at(slot_of(b + y), a, tile, NW, w, j) + l] = (f32x4){h[0], h[1], h[2], h[3]};
        join_step<INF>(h, A2, d[y], c[y], x[y]);
      }
    }
  };
  if (__builtin_amdgcn_ballot_w64(sInf[min(l, waves - 1)] != 0)) hand_on(std::true_type());
  else hand_on(std::false_type());
}

// ------------------------------------------------------------------------------------------------ backward
constexpr int kSub = 2;   // tokens whose decays and states are in registers

template <typename T, int NW, bool FULL>
__global__ __launch_bounds__(64 * NW, 2) void scan_bwd_kernel(ScanArgs a) {
  constexpr int kOwn = (4 + NW - 1) / NW;   // arrays that a wave fetches for the workgroup
  __shared__ float sBC[NW][kTok][2][16];
  __shared__ __attribute__((aligned(16))) T sRow[4][kTok][64];   // u, delta, z, dy; then du, ddelta, dz in the places of the first three
  __shared__ float sDt[kTok][64];
  __shared__ f32x4 sH[NW][kTok / kSub - 1][4][64];
  __shared__ __attribute__((aligned(16))) float sP[NW][kTok][32];   // the waves' shares of dB and dC
  __shared__ float sS[NW > 1 ? 2 : 1][NW > 1 ? NW : 1][kSub][3][64];
  Lane ln(a);
  if (NW == 1) ln.w = 0;      // (known to the compiler)
  const int l = threadIdx.x & 63, w = ln.w, row = ln.row, own = own_at();
  const int t0 = blockIdx.y * a.seg, t1 = min(a.T, t0 + a.seg);
  const float bias = a.bias && ln.on ? a.bias[ln.own] : 0.f, Dc = a.D ? a.D[ln.own] : 0.f;
  float A2[4][4], carry[4][4], dA[4][4];
  float dD = 0.f, dbias = 0.f;
  ln.load(a, a.A, A2);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[k][i] *= kLog2e;
  zero44(dA);
  const bool beyond = !FULL && 16 * (w + 1) > a.N;      // entries beyond N in this wave
  const int64_t slot = (int64_t)row * a.segs + blockIdx.y;
  if (t1 < a.T) load_packed(ln, a.seg_h, packed_at(slot, a, ln.tile, NW, w, 0), carry);
  else zero44(carry);
  if (beyond) ln.clear_beyond(a, carry);
  ScanSeq cur = seq_at(a, row, t1 - 1);
  if (t1 == a.T && a.cu) hand_over(a, ln, a.d_final, a.d_init, cur.n + 1, a.seqs);   // sequences without a token behind the last one
  const int64_t out0 = (int64_t)row * a.T * a.D_;
  const int shares = ((l >> 4) & 1) * 16 + 4 * (l & 3) + ((l >> 2) & 1) * 2 + ((l >> 3) & 1);   // a lane's sum among dB and dC (below)
  const bool has_z = a.z != nullptr;
  int turn = 0;
  auto sync = [&]() {
    if constexpr (NW == 1) wave_lds_fence();
    else __syncthreads();
  };

  const T* pB = (const T*)a.Bm + row * a.Bb + (int64_t)ln.group * a.N;
  const T* pC = (const T*)a.Cm + row * a.Cb + (int64_t)ln.group * a.N;
  const int n4 = 16 * w + 4 * (l & 3);
  BlockRows<T> rows[kOwn];
  Four<T> rb, rc;
  float h0[4][4];              // the state kept before the block
  auto fetch = [&](int tb) {
    const int left = min(kTok, t1 - tb) - 1;
#pragma unroll
    for (int m = 0; m < kOwn; ++m) {
      const int i = w + NW * m;
      if (i > 3 || (i == 2 && !a.z)) continue;
      const T* p = (const T*)(i == 0 ? a.u : i == 1 ? a.delta : i == 2 ? a.z : a.dy);
      const int64_t batch = i == 0 ? a.ub : i == 1 ? a.db : i == 2 ? a.zb : (int64_t)a.T * a.D_;
      const int stride = i == 0 ? a.ut : i == 1 ? a.dt : i == 2 ? a.zt : a.D_;
      rows[m].fetch(ln, p + row * batch + (int64_t)tb * stride, stride, left);
    }
    const int t = min((l >> 2) & 7, left);
    rb.fetch(a, pB + (int64_t)tb * a.Bt, __umul24(t, a.Bt) * (unsigned)sizeof(T), n4);
    rc.fetch(a, pC + (int64_t)tb * a.Ct, __umul24(t, a.Ct) * (unsigned)sizeof(T), n4);
  };
  auto fetch_kept = [&](int tb) { load_packed(ln, a.ckpt, packed_at((int64_t)row * a.ckpts + tb / kTok, a, ln.tile, NW, w, 0), h0); };
  // results of a block: out of LDS, and on their way
  BlockRows<T> done[kOwn];
  f32x4 done_bc;
  auto take = [&]() {
#pragma unroll
    for (int m = 0; m < kOwn; ++m) done[m].from_lds(sRow[min(w + NW * m, 2)]);
    done_bc = *(const f32x4*)&sP[w][l >> 3][4 * (l & 7)];
  };
  auto put = [&](int tb, int nt) {
#pragma unroll
    for (int m = 0; m < kOwn; ++m) {
      const int i = w + NW * m;
      if (i > 2 || (i == 2 && !a.z)) continue;
      done[m].store(ln, (T*)(i == 0 ? a.du : i == 1 ? a.ddelta : a.dz) + out0 + (int64_t)tb * a.D_, a.D_, nt);
    }
    const float* to = a.part_bc + ((((int64_t)row * a.T + tb) * a.tiles + ln.tile) * NW + w) * 32;
    if ((l >> 3) < nt) *(PAL_GLOBAL f32x4*)row_element(to, ((l >> 3) * a.tiles * NW * 32 + 4 * (l & 7)) * 4u) = done_bc;
  };
  const int last = t0 + (t1 - 1 - t0) / kTok * kTok;
  fetch(last);
  fetch_kept(last);

  for (int tb = last; tb >= t0; tb -= kTok) {
    const int nt = min(kTok, t1 - tb);
    // ---- the block's rows, time steps, and its states before tokens 2, 4 and 6
    take();     // (before the first block: nothing, and it goes nowhere)
    sync();
#pragma unroll
    for (int m = 0; m < kOwn; ++m) {
      const int i = w + NW * m;
      if (i <= 3) rows[m].to_lds(sRow[i]);
    }
    *(f32x4*)&sBC[w][(l >> 2) & 7][0][4 * (l & 3)] = rb.get(a, n4);
    *(f32x4*)&sBC[w][(l >> 2) & 7][1][4 * (l & 3)] = rc.get(a, n4);
    settle44(h0);      // (older than the next fetch: waited for behind it, it would take that with it)
    sync();
    // (the stores after the wait for this block's rows and before the next fetch: they are never waited for by themselves)
    if (tb < last) put(tb + kTok, min(kTok, t1 - tb - kTok));
    if (tb > t0) fetch(tb - kTok);
    {
      constexpr int K = (kTok + NW - 1) / NW;      // tokens of a wave (three waves: one token twice)
      const int first = min(K * w, kTok - K);
      float raw[K], dt[K];
#pragma unroll
      for (int i = 0; i < K; ++i) raw[i] = to_f32(sRow[1][first + i][own]) + bias;
      stage();
      time_steps<T, K>(raw, dt, a.softplus);
#pragma unroll
      for (int i = 0; i < K; ++i) sDt[first + i][l] = dt[i];
    }
    sync();
    // A whole block in which no sequence starts or ends is straight code: one path for the registers that are carried from block to
    // block.  (Loops around it, over parts and over pairs of tokens, moved them, 16 states, 16 decays' gradients and the 16 states on
    // their way from memory, between two sets on every round, and waited for the last.)
    bool clear = false;
    if (beyond) {
      float most = 0.f;
#pragma unroll
      for (int t = 0; t < kTok; ++t) {
        const float dt = sDt[t][l], gy = to_f32(sRow[3][t][own]) * (has_z ? to_f32(sRow[2][t][own]) : 1.f);   // (at least |dy silu(z)|)
        most = fmaxf(fmaxf(fmaxf(most, fabsf(dt)), fabsf(dt * to_f32(sRow[0][t][own]))), fabsf(gy));
      }
      clear = any_infinite(most);
    }
    const bool plain = nt == kTok && cur.s < tb && cur.e > tb + kTok && !clear;
    auto states = [&](auto kind) __attribute__((always_inline)) {
      float h[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) h[k][i] = h0[k][i];
      auto walk = [&](auto r) {
#pragma unroll
        for (int t = 0; t < kTok - kSub; ++t) {
          if (walks(r, t)) {
            const float dt = sDt[t][l], x = dt * to_f32(sRow[0][t][own]);
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
          }
        }
      };
      if constexpr (decltype(kind)::whole) {
        walk(kind);
      } else {
        const int most = min(nt, kTok - kSub);
        ScanSeq fw = seq_at(a, row, tb);     // (`cur` where that is the one would put it into memory, for the choice between two addresses)
        for (int lo = 0, hi; lo < most; lo = hi) {
          if (tb + lo == fw.s) load_state(a, ln, a.init, fw.n, h);
          hi = max(lo + 1, min(most, fw.e - tb));
          walk(Part{lo, hi});
          if (hi < most) fw = next_seq(a, fw);
        }
      }
    };
    // ---- two tokens at a time from the end
    auto pair = [&](auto kind, int sub) __attribute__((always_inline)) {
      constexpr bool whole = decltype(kind)::whole;
      const int ts = tb + sub * kSub, ns = whole ? kSub : min(kSub, t1 - ts);
      // what the tokens take and, in the same place, what they give once they are done: Y -> du, slope (of the softplus) -> ddelta,
      // gz (dy silu'(z)) -> dz
      float uv[kSub], Y[kSub], slope[kSub], gz[kSub];
      float x2[2 * kSub], sg[2 * kSub];      // raw time steps and gates (without z: whatever is there, and not used)
#pragma unroll
      for (int t = 0; t < kSub; ++t) {
        x2[t] = to_f32(sRow[1][sub * kSub + t][own]) + bias;
        x2[kSub + t] = to_f32(sRow[2][sub * kSub + t][own]);
        uv[t] = to_f32(sRow[0][sub * kSub + t][own]);
        Y[t] = to_f32(sRow[3][sub * kSub + t][own]);
      }
      stage();
      sigmoids<T, 2 * kSub>(x2, sg);
#pragma unroll
      for (int t = 0; t < kSub; ++t) {
        slope[t] = a.softplus && x2[t] <= 20.f ? sg[t] : 1.f;
        const float z = x2[kSub + t], s = sg[kSub + t];
        gz[t] = has_z ? Y[t] * (s + z * s * (1.f - s)) : 0.f;
        Y[t] *= has_z ? z * s : 1.f;
      }
      auto finish = [&](int t, float dt, float ypre, float sumB, float sumA) {
        const float ddt = fmaf(uv[t], sumB, sumA * 0.6931471806f);
        gz[t] *= fmaf(Dc, uv[t], ypre);
        dD = fmaf(Y[t], uv[t], dD);
        slope[t] *= ddt;
        dbias += slope[t];
        Y[t] = fmaf(dt, sumB, Dc * Y[t]);
        sRow[0][sub * kSub + t][own] = from_f32<T>(Y[t]);
        sRow[1][sub * kSub + t][own] = from_f32<T>(slope[t]);
        sRow[2][sub * kSub + t][own] = from_f32<T>(gz[t]);
      };
      float h[4][4];
      auto walk = [&](auto r, bool ends) __attribute__((always_inline)) {
        float av[kSub][4][4], ah[kSub][4][4];
        const int have = !FULL && !whole && clear ? ln.entries(a) : 4;      // entries that count in the sums over n
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
          if (!walks(r, t)) continue;
          const float dt = sDt[sub * kSub + t][l], x = dt * uv[t];
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
        }
        if constexpr (whole) {
          if (sub == 0) {      // h0 is used up: the next block's (or the last one's again), while the last two tokens of this one are walked
            stage();
            fetch_kept(max(tb - kTok, t0));
          }
        } else if (ends) {
          load_state(a, ln, a.d_final, cur.n, carry);
        }
#pragma unroll
        for (int t = kSub - 1; t >= 0; --t) {
          if (!walks(r, t)) continue;
          const float dt = sDt[sub * kSub + t][l], x = dt * uv[t];
          const f32x4 Bv = *(const f32x4*)&sBC[w][sub * kSub + t][0][4 * ln.j];
          const f32x4 Cv = *(const f32x4*)&sBC[w][sub * kSub + t][1][4 * ln.j];
          const float dk[4] = {of_channel<0>(dt), of_channel<1>(dt), of_channel<2>(dt), of_channel<3>(dt)};
          const float xk[4] = {of_channel<0>(x), of_channel<1>(x), of_channel<2>(x), of_channel<3>(x)};
          const float Yk[4] = {of_channel<0>(Y[t]), of_channel<1>(Y[t]), of_channel<2>(Y[t]), of_channel<3>(Y[t])};
          float gB[4], gC[4], sy[4], sb[4], sa[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float hv = fmaf(xk[k], Bv[i], ah[t][k][i]), g = fmaf(Cv[i], Yk[k], carry[k][i]);
              float p = g * ah[t][k][i];
              carry[k][i] = g * av[t][k][i];
              if (!FULL && !whole && i >= have) hv = g = p = 0.f;
              gC[i] = k ? fmaf(Yk[k], hv, gC[i]) : Yk[k] * hv;
              gB[i] = k ? fmaf(g, xk[k], gB[i]) : g * xk[k];
              sy[k] = i ? fmaf(Cv[i], hv, sy[k]) : Cv[i] * hv;
              sb[k] = i ? fmaf(g, Bv[i], sb[k]) : g * Bv[i];
              sa[k] = i ? fmaf(p, A2[k][i], sa[k]) : p * A2[k][i];
              dA[k][i] = fmaf(p, dk[k], dA[k][i]);
            }
          }
          // dB, dC: eight sums over the sixteen quads; lane bits 3, 2, 4 choose among them, bit 5 holds the same twice
          {
            const float p0 = pair_bit3(gB[0], gB[1]), p1 = pair_bit3(gB[2], gB[3]);
            const float p2 = pair_bit3(gC[0], gC[1]), p3 = pair_bit3(gC[2], gC[3]);
            float r0 = pair_bit2(p0, p1), r1 = pair_bit2(p2, p3);
            swap_rows(r0, r1);
            float s = r0 + r1, s2 = s;
            swap_halves(s, s2);
            sP[w][sub * kSub + t][shares] = s + s2;
          }
          const float ty = quad_total4(sy[0], sy[1], sy[2], sy[3], ln.odd, ln.high);
          const float tB = quad_total4(sb[0], sb[1], sb[2], sb[3], ln.odd, ln.high);
          const float tA = quad_total4(sa[0], sa[1], sa[2], sa[3], ln.odd, ln.high);
          if constexpr (NW == 1) {
            finish(t, dt, ty, tB, tA);
          } else {
            sS[turn][w][t][0][l] = ty;
            sS[turn][w][t][1][l] = tB;
            sS[turn][w][t][2][l] = tA;
          }
        }
      };
      auto start = [&]() {      // the state before the pair
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f32x4 v = sub ? sH[w][max(sub - 1, 0)][k][l] : (f32x4){h0[k][0], h0[k][1], h0[k][2], h0[k][3]};
#pragma unroll
          for (int i = 0; i < 4; ++i) h[k][i] = v[i];
        }
      };
      if constexpr (whole) {
        start();
        walk(kind, false);
        settle44(dA);       // (or the sums of all pairs are put off to the last one, and what goes into them is kept)
      } else {
        for (int hi = ns, lo; hi > 0; hi = lo) {
          lo = min(hi - 1, max(0, cur.s - ts));
          if (ts + lo == cur.s) load_state(a, ln, a.init, cur.n, h);
          else start();
          walk(Part{lo, hi}, ts + hi == cur.e);
          if (ts + lo == cur.s) {
            if (a.d_init) store_state(a, ln, a.d_init, cur.n, carry);
            if (a.cu) {
              const ScanSeq prev = prev_seq(a, cur);
              hand_over(a, ln, a.d_final, a.d_init, prev.n + 1, cur.n);
              cur = prev;
            }
          }
        }
      }
      if constexpr (NW > 1) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
          if ((sub * kSub + t) % NW != w || t >= ns) continue;
          float s3[3];
#pragma unroll
          for (int x = 0; x < 3; ++x) {
            s3[x] = sS[turn][0][t][x][l];
#pragma unroll
            for (int k = 1; k < NW; ++k) s3[x] += sS[turn][k][t][x][l];
          }
          finish(t, sDt[sub * kSub + t][l], s3[0], s3[1], s3[2]);
        }
        turn ^= 1;
      }
    };
    if (plain) {
      states(Whole{0, 0});
      wave_lds_fence();
#pragma unroll
      for (int sub = kTok / kSub - 1; sub >= 0; --sub) pair(Whole{0, 0}, sub);
    } else {
      states(Part{0, 0});
      wave_lds_fence();
      for (int sub = (nt - 1) / kSub; sub >= 0; --sub) pair(Part{0, 0}, sub);
      if (!FULL && clear) ln.clear_beyond(a, carry);
      fetch_kept(max(tb - kTok, t0));
      settle44(h0);
    }
    sync();
  }
  take();
  put(t0, min(kTok, t1 - t0));
  store_packed(ln, a.part_a, packed_at(slot, a, ln.tile, NW, w, 0), dA);
  float* pc = a.part_c + (((slot * a.tiles + ln.tile) * NW + w) * 64 + l) * 2;
  pc[0] = dD;
  pc[1] = dbias;
}

// dB, dC [rows, T, G, N]: the tiles of a group in their order.  Thread = four entries of a token.
template <typename T>
__device__ __forceinline__ void sum_rows(const ScanArgs& a, int nw, int64_t first, int64_t step) {
  const int64_t per = 2 * (int64_t)a.G * nw * 4, total = (int64_t)a.rows * a.T * per;
  for (int64_t x = first; x < total; x += step) {
    const int64_t tok = x / per;
    const int r = (int)(x - tok * per), j = r & 3, which = (r >> 2) & 1, w = (r >> 3) % nw, g = (r >> 3) / nw, n = 16 * w + 4 * j;
    const f32x4* p = (const f32x4*)(a.part_bc + ((tok * a.tiles + (int64_t)g * a.tiles_g) * nw + w) * 32 + which * 16 + 4 * j);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < a.tiles_g; i0 += 8) {
      f32x4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[(int64_t)min(i0 + i, a.tiles_g - 1) * nw * 8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < a.tiles_g) s += v[i];
    }
    T* out = (T*)(which ? a.dC : a.dB) + (tok * a.G + g) * a.N + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) out[i] = from_f32<T>(s[i]);
  }
}

// dA, dD, ddelta_bias: the segments of all rows in their order, in 64 bits.  Workgroup = a tile, one of its waves and z: z < 4 the entries
// 4 z .. of dA, z = 4 dD and ddelta_bias; sixteen waves take a share of the segments each.  Behind these workgroups those of dB and dC, in one
// launch.
constexpr int kSumWaves = 16;
template <typename T>
__global__ __launch_bounds__(64 * kSumWaves) void scan_bwd_sums_kernel(ScanArgs a, int nw) {
  __shared__ double s[kSumWaves][64][4];
  const int first = a.tiles * nw * 5;
  if ((int)blockIdx.x >= first) {
    sum_rows<T>(a, nw, (int64_t)(blockIdx.x - first) * (64 * kSumWaves) + threadIdx.x, (int64_t)(gridDim.x - first) * (64 * kSumWaves));
    return;
  }
  const int l = threadIdx.x & 63, v = threadIdx.x >> 6, z = blockIdx.x % 5, tile = blockIdx.x / 5 / nw, w = blockIdx.x / 5 - tile * nw;
  const int64_t slots = (int64_t)a.rows * a.segs;
  const int group = tile / a.tiles_g, base = group * a.per_group + (tile - group * a.tiles_g) * 64, end = (group + 1) * a.per_group;
  double t[4] = {0., 0., 0., 0.};
  if (z < 4) {
#pragma unroll 4
    for (int64_t i = v; i < slots; i += kSumWaves) {
      const f32x4 x = ((const f32x4*)a.part_a)[packed_at(i, a, tile, nw, w, z) + l];
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] += x[e];
    }
  } else if (w == 0) {
#pragma unroll 4
    for (int64_t q = v; q < slots * nw; q += kSumWaves) {
      const int64_t i = q / nw, k = q - i * nw;
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
  for (int e = 0; e < 4; ++e) {
    t[e] = 0.;
    for (int x = 0; x < kSumWaves; ++x) t[e] += s[x][l][e];
  }
  if (z < 4) {
    const int c = base + l, n0 = 16 * w + 4 * z;
    if (c < end)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n0 + e < a.N) a.dA[(int64_t)c * a.N + n0 + e] = (float)t[e];
  } else if (w == 0) {
    const int c = base + 16 * (l & 3) + (l >> 2);
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
  if (d->batch > 65535 || d->channels >= 1 << 24 || d->channels % d->groups) return PAL_E_DIM;
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
  for (int64_t s : {d->u_token, d->delta_token, d->z_token, d->B_token, d->C_token})
    if (s >= 1 << 24) return PAL_E_DIM;
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

// Tokens per segment: enough segments for `most` waves, at least 32 tokens each.  Forward three waves on every SIMD (1 x 16384 tokens of 1536
// channels: 114 us with three, 131 with two, 116 with four), backward the two whose registers fit.  (4096 tokens of 384 channels in two
// groups, all kernels of a forward and backward: segments of at least 64 tokens 270 us, of 32 183, of 16 181.)
constexpr int64_t kSimds = 1024;   // of the GPU
static int scan_segment(const PalScanDims* d, int64_t most) {
  const int64_t waves = scan_tiles(d) * scan_waves(d) * d->batch;
  const int64_t segs = waves < most ? most / waves : 1;
  int64_t seg = (d->seq_len + segs - 1) / segs;
  seg = (seg + PAL_SCAN_BLOCK - 1) / PAL_SCAN_BLOCK * PAL_SCAN_BLOCK;
  if (seg < 32) seg = 32;
  return (int)(seg < d->seq_len ? seg : (d->seq_len + PAL_SCAN_BLOCK - 1) / PAL_SCAN_BLOCK * PAL_SCAN_BLOCK);
}
static void scan_args(ScanArgs& a, const PalScanDims* d, const PalScanTensors* t, bool back) {
  a.rows = d->batch; a.T = d->seq_len; a.seqs = d->n_seqs; a.D_ = d->channels; a.N = d->state; a.G = d->groups;
  a.per_group = d->channels / d->groups;
  a.tiles_g = (a.per_group + 63) / 64;
  a.tiles = a.G * a.tiles_g;
  a.softplus = d->softplus;
  a.vec = d->state % 4 == 0;
  a.ub = d->u_batch; a.db = d->delta_batch; a.zb = d->z_batch; a.Bb = d->B_batch; a.Cb = d->C_batch;
  a.ut = (int)d->u_token; a.dt = (int)d->delta_token; a.zt = (int)d->z_token; a.Bt = (int)d->B_token; a.Ct = (int)d->C_token;
  a.seg = scan_segment(d, (back ? 2 : 3) * kSimds);
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

// waves over the segments of a join: a batch of loads each, up to kJoinWaves
static int join_waves(const ScanArgs& a) {
  const int w = (a.segs + kJoinAhead - 1) / kJoinAhead;
  return w < kJoinWaves ? w : kJoinWaves;
}
template <typename T, int LPC>
static int scan_step_run(const ScanArgs& a, hipStream_t s) {
  const int per = 256 / LPC;
  PAL_TIMED_LAUNCH(kKernScanFwd, s, (scan_step_kernel<T, LPC>), dim3((a.D_ + per - 1) / per, a.rows), dim3(256), 0, s, a);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
template <typename T, int NW, bool FULL>
static int scan_fwd_run(const ScanArgs& a, hipStream_t s) {
  const dim3 grid(a.tiles, a.segs, a.rows);
  if (a.segs > 1) {
    PAL_TIMED_LAUNCH(kKernScanSegment, s, (scan_fwd_kernel<T, NW, false, true>), grid, dim3(64 * NW), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
    PAL_TIMED_LAUNCH(kKernScanJoin, s, (scan_join_kernel<NW, false>), dim3(a.tiles, 4 * NW, a.rows), dim3(64 * join_waves(a)), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
  }
  PAL_TIMED_LAUNCH(kKernScanFwd, s, (scan_fwd_kernel<T, NW, true, FULL>), grid, dim3(64 * NW), 0, s, a);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
template <typename T, int NW, bool FULL>
static int scan_bwd_run(const ScanArgs& a, hipStream_t s) {
  const dim3 grid(a.tiles, a.segs, a.rows);
  if (a.segs > 1) {
    PAL_TIMED_LAUNCH(kKernScanSegment, s, (scan_back_segment_kernel<T, NW>), grid, dim3(64 * NW), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
    PAL_TIMED_LAUNCH(kKernScanJoin, s, (scan_join_kernel<NW, true>), dim3(a.tiles, 4 * NW, a.rows), dim3(64 * join_waves(a)), 0, s, a);
    PAL_HIP_LAUNCH_CHECK();
  }
  PAL_TIMED_LAUNCH(kKernScanBwd, s, (scan_bwd_kernel<T, NW, FULL>), grid, dim3(64 * NW), 0, s, a);
  PAL_HIP_LAUNCH_CHECK();
  const int64_t n = 8 * (int64_t)a.rows * a.T * a.G * NW, blocks = (n + 64 * kSumWaves - 1) / (64 * kSumWaves);
  PAL_TIMED_LAUNCH(kKernScanBwdSums, s, scan_bwd_sums_kernel<T>, dim3(a.tiles * NW * 5 + (unsigned)(blocks < 2048 ? blocks : 2048)),
                   dim3(64 * kSumWaves), 0, s, a, NW);
  PAL_HIP_LAUNCH_CHECK();
  return PAL_OK;
}
template <typename T>
static int scan_fwd_waves(const ScanArgs& a, int nw, hipStream_t s) {
  if (a.T <= kStepTokens && !a.cu && !a.ckpt) {
    if (a.N == 4) return scan_step_run<T, 1>(a, s);
    if (a.N == 8) return scan_step_run<T, 2>(a, s);
    if (a.N == 16) return scan_step_run<T, 4>(a, s);
    if (a.N == 32) return scan_step_run<T, 8>(a, s);
    if (a.N == 64) return scan_step_run<T, 16>(a, s);
  }
  switch (nw) {
    case 1: return a.N % 16 ? scan_fwd_run<T, 1, false>(a, s) : scan_fwd_run<T, 1, true>(a, s);
    case 2: return a.N % 16 ? scan_fwd_run<T, 2, false>(a, s) : scan_fwd_run<T, 2, true>(a, s);
    case 3: return a.N % 16 ? scan_fwd_run<T, 3, false>(a, s) : scan_fwd_run<T, 3, true>(a, s);
    default: return a.N % 16 ? scan_fwd_run<T, 4, false>(a, s) : scan_fwd_run<T, 4, true>(a, s);
  }
}
template <typename T>
static int scan_bwd_waves(const ScanArgs& a, int nw, hipStream_t s) {
  switch (nw) {
    case 1: return a.N % 16 ? scan_bwd_run<T, 1, false>(a, s) : scan_bwd_run<T, 1, true>(a, s);
    case 2: return a.N % 16 ? scan_bwd_run<T, 2, false>(a, s) : scan_bwd_run<T, 2, true>(a, s);
    case 3: return a.N % 16 ? scan_bwd_run<T, 3, false>(a, s) : scan_bwd_run<T, 3, true>(a, s);
    default: return a.N % 16 ? scan_bwd_run<T, 4, false>(a, s) : scan_bwd_run<T, 4, true>(a, s);
  }
}

}  // namespace pal

extern "C" size_t pal_scan_checkpoint_bytes(const PalScanDims* d) {
  using namespace pal;
  if (check_scan(d) != PAL_OK) return 0;
  ScanArgs a{};
  scan_args(a, d, nullptr, false);
  return packed_bytes(a, scan_waves(d), (int64_t)a.rows * a.ckpts);
}

extern "C" size_t pal_scan_fwd_workspace_bytes(const PalScanDims* d) {
  using namespace pal;
  if (check_scan(d) != PAL_OK) return 0;
  ScanArgs a{};
  scan_args(a, d, nullptr, false);
  return a.segs > 1 ? seg_bytes(a, scan_waves(d)) : 0;
}

extern "C" int pal_scan_fwd(const PalScanDims* d, const PalScanTensors* t, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace pal;
  if (int rc = check_scan(d)) return rc;
  if (int rc = check_scan_tensors(d, t)) return rc;
  if (!t->y) return PAL_E_NULL;
  if (((d->flags & PAL_FLAG_STORE_FINAL) != 0) != (t->final_ != nullptr)) return PAL_E_STATE;
  if (t->cu_seqlens && t->final_ && t->final_ == t->init) return PAL_E_STATE;   // read by one segment, written by another
  ScanArgs a{};
  scan_args(a, d, t, false);
  const int nw = scan_waves(d);
  if (a.segs > 65535 || (int64_t)a.tiles * nw > 1 << 20) return PAL_E_DIM;   // (the second: the threads of a launch, and 32-bit places)
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
  scan_args(a, d, nullptr, true);
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
  scan_args(a, d, t, true);
  const int nw = scan_waves(d);
  // (the second: 32-bit places in a block's shares, and the threads of the sums, which have five workgroups of 1024 for each)
  if (a.segs > 65535 || (int64_t)a.tiles * nw > 1 << 19) return PAL_E_DIM;
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
