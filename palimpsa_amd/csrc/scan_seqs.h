// The sequences of a packed batch as the selective scan walks through them: forward from the one that holds a token to the next that has
// any, backward to the one before.  Args: cu (bounds, NULL for a dense batch), seqs (their number) and T (tokens of a row).
#pragma once
#include <cstdint>

namespace pal {

// a sequence: its number and its tokens [s, e) in the row
struct ScanSeq {
  int n, s, e;
};
// Bounds are held to the tokens of the row, and what comes before the first and behind the last sequence starts and ends at no token: an
// array that does not ascend from 0 to T cannot make a kernel read or write a state that is not there (results are then unspecified).
template <typename Args>
__device__ __forceinline__ int seq_bound(const Args& a, int i) { return min(max(a.cu[i], 0), a.T); }
template <typename Args>
__device__ __forceinline__ ScanSeq seq_at(const Args& a, int row, int t) {
  if (!a.cu) return {row, 0, a.T};
  int lo = 0, hi = a.seqs - 1;      // last sequence that starts at t or before: it holds t if any does
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return {lo, seq_bound(a, lo), seq_bound(a, lo + 1)};
}
// the sequence after / before `s` that has a token
template <typename Args>
__device__ __forceinline__ ScanSeq next_seq(const Args& a, const ScanSeq& s) {
  int n = s.n + 1;
  while (n < a.seqs && seq_bound(a, n + 1) <= s.e) ++n;
  return n < a.seqs ? ScanSeq{n, s.e, seq_bound(a, n + 1)} : ScanSeq{a.seqs, a.T + 1, a.T + 1};
}
template <typename Args>
__device__ __forceinline__ ScanSeq prev_seq(const Args& a, const ScanSeq& s) {
  int n = s.n - 1;
  while (n >= 0 && seq_bound(a, n) >= s.s) --n;
  return n >= 0 ? ScanSeq{n, seq_bound(a, n), s.s} : ScanSeq{-1, -1, -1};
}

}  // namespace pal
