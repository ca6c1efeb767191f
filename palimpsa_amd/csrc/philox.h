// Random words of a dropout, by counter: Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with
// seven rounds, the fewest that the authors found to pass every test.  A word is a function of its place and the seed alone, so a
// backward pass makes the same ones again and nothing is stored.  Ten rounds would be 20 wide products for four words instead of 14, at a quarter
// of the rate of other instructions: they are the larger part of a dropout's time in the vector units.
#pragma once
#include "pal_common.h"

namespace pal {

struct DropArgs {
  const int64_t* seed_at;
  uint64_t seed;
  uint32_t site;
  uint32_t least;    // a word that is kept is not below
  float scale;       // 1 / (1 - p)
};

struct DropKey {
  uint32_t k0, k1;
  __device__ __forceinline__ explicit DropKey(const DropArgs& d) {
    const uint64_t s = d.seed_at ? (uint64_t)*d.seed_at : d.seed;
    k0 = __builtin_amdgcn_readfirstlane((uint32_t)s);
    k1 = __builtin_amdgcn_readfirstlane((uint32_t)(s >> 32));
  }
};

// the words of columns 4 q .. of a row
__device__ __forceinline__ void drop_words(uint32_t (&w)[4], uint32_t q, int64_t row, const DropArgs& d, DropKey key) {
  uint32_t c0 = q, c1 = (uint32_t)row, c2 = (uint32_t)((uint64_t)row >> 32), c3 = d.site;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ key.k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ key.k1;
    c3 = (uint32_t)a;
    key.k0 += 0x9E3779B9u;
    key.k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}
// entries 8 piece .. of a row: kept ones times the scale, zero for the others (whatever they hold)
__device__ __forceinline__ void drop_piece(float* x, uint32_t piece, int64_t row, const DropArgs& d, const DropKey& key) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
    drop_words(w, 2 * piece + h, row, d, key);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * h + e] = w[e] >= d.least ? x[4 * h + e] * d.scale : 0.f;
  }
}

// host: PAL_OK and the kernels' form of a dropout, or an error code; p = 0 has no form of its own
inline int drop_args(const PalDropout& p, DropArgs& d) {
  if (!(p.p >= 0.0) || !(p.p < 1.0)) return PAL_E_DIM;
  d.seed_at = p.p > 0.0 ? p.seed_at : nullptr;
  d.seed = (uint64_t)p.seed;
  d.site = p.site;
  const double least = p.p * 4294967296.0;
  const uint64_t n = (uint64_t)least, up = least - (double)n >= 0.5;
  d.least = n + up > 0xffffffffull ? 0xffffffffu : (uint32_t)(n + up);
  d.scale = (float)(1.0 / (1.0 - p.p));
  return PAL_OK;
}

}  // namespace pal
