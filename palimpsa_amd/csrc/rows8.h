// Rows of any length and alignment, eight consecutive elements per lane: whole pieces move as 16-byte accesses (which the
// global memory path takes at any element's address), the last piece of a row whose length is no multiple of eight
// element by element.
#pragma once
#include <type_traits>

#include "pal_common.h"

namespace pal {

typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// eight elements as fetched, converted when they are used
template <typename T>
struct Piece8;
template <>
struct Piece8<bf16_t> {
  bf16x8 v;
  __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
  __device__ __forceinline__ bf16_t at(int e) const { return v[e]; }
  __device__ __forceinline__ void set(int e, bf16_t x) { v[e] = x; }
  template <typename P>   // (pointers of any address space)
  __device__ __forceinline__ void load(P p) { v = *(const __attribute__((address_space(1))) bf16x8_any*)p; }
  template <typename P>
  __device__ __forceinline__ void store(P p) const { *(__attribute__((address_space(1))) bf16x8_any*)p = v; }
  // a use of the value: whoever loaded it waits here
  __device__ __forceinline__ void settle() {
    f32x4 x = __builtin_bit_cast(f32x4, v);
    asm volatile("" : "+v"(x));
    v = __builtin_bit_cast(bf16x8, x);
  }
};
template <>
struct Piece8<float> {
  f32x4 lo, hi;
  __device__ __forceinline__ float get(int e) const { return e < 4 ? lo[e & 3] : hi[e & 3]; }
  __device__ __forceinline__ float at(int e) const { return get(e); }
  __device__ __forceinline__ void set(int e, float x) { if (e < 4) lo[e & 3] = x; else hi[e & 3] = x; }
  template <typename P>
  __device__ __forceinline__ void load(P p) {
    lo = *(const __attribute__((address_space(1))) f32x4_any*)p;
    hi = *(const __attribute__((address_space(1))) f32x4_any*)(p + 4);
  }
  template <typename P>
  __device__ __forceinline__ void store(P p) const {
    *(__attribute__((address_space(1))) f32x4_any*)p = lo;
    *(__attribute__((address_space(1))) f32x4_any*)(p + 4) = hi;
  }
  __device__ __forceinline__ void settle() { asm volatile("" : "+v"(lo), "+v"(hi)); }
};

// `n` elements of the piece are there (8 or more: all; 0 or less: none, and nothing is read), the others are zero
template <typename T>
__device__ __forceinline__ void load_piece(Piece8<T>& d, const T* p, int n) {
  if (n >= 8) {
    d.load(p);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) d.set(e, e < n ? p[e] : (T)0.f);
  }
}
__device__ __forceinline__ void store_piece(bf16_t* p, const float* x, int n) {
  if (n >= 8) {
    const bf16x2 a = pack2(x[0], x[1]), b = pack2(x[2], x[3]), c = pack2(x[4], x[5]), d = pack2(x[6], x[7]);
    const bf16x8 v = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    *(bf16x8_any*)p = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (bf16_t)x[e];
  }
}
__device__ __forceinline__ void store_piece(float* p, const float* x, int n) {
  if (n >= 8) {
    const f32x4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
    *(f32x4_any*)p = a;
    *(f32x4_any*)(p + 4) = b;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = x[e];
  }
}

// eight per-channel parameters of either type; whichever it is, they are waited for in their branch (where the two meet, the
// compiler would wait for everything in flight)
__device__ __forceinline__ void load_params(float* x, const void* p, int64_t i, int is_bf16) {
  if (is_bf16) {
    const bf16x8 v = *(const bf16x8_any*)((const bf16_t*)p + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
  } else {
    const f32x4 lo = *(const f32x4_any*)((const float*)p + i), hi = *(const f32x4_any*)((const float*)p + i + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < 4 ? lo[e & 3] : hi[e & 3];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(x[e]));
}
// the same of fewer: those beyond n zero
__device__ __forceinline__ void load_few_params(float* x, const void* p, int is_bf16, int n) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e < n ? load_rt(p, e, is_bf16) : 0.f;
}

// logistic function by the one-instruction reciprocal (1 ulp; an IEEE division is ten instructions)
__device__ __forceinline__ float logistic(float x) { return fast_rcp(1.f + __expf(-x)); }

}  // namespace pal
