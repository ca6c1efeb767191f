// What the norms of rows share: how a row lies in the registers of a wave or of four, and sums over it.
#pragma once
#include "rows8.h"

namespace pal {

constexpr int kNormMaxRow = 16384;

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

}  // namespace pal
