// Sequences of a flat axis of tokens, as the convolution and the selective scan walk it.
#pragma once

#include <hip/hip_runtime.h>

namespace ltc {

// The sequence of a token: tokens lo up to hi. s < 0: the token lies outside all
// sequences, and so do those up to hi.
struct Seq {
  int s, lo, hi;
  long long off;  // what a sequence adds to the offset t * st of token t
};

// Sequence of token t < N: of batches of T steps (cu null), or of S packed sequences.
// Boundaries of any values and order give lo <= t < hi within 0 ... N: the search ends
// with cu[s] <= t < cu[s + 1].
__device__ __forceinline__ Seq seq_of(const int* cu, int S, int T, int N, int t, long long sb, long long st) {
  Seq q;
  if (cu == nullptr) {
    q.s = (int)((unsigned)t / (unsigned)T);
    q.lo = q.s * T;
    q.hi = q.lo + T;
    q.off = q.s * sb - q.lo * st;
    return q;
  }
  int a = 0, b = S + 1;
  while (a < b) {
    const int mid = (int)(((unsigned)a + (unsigned)b) / 2);
    if (cu[mid] <= t) a = mid + 1;
    else b = mid;
  }
  q.s = a - 1 < S ? a - 1 : -1;
  q.lo = a > 0 ? max(cu[a - 1], 0) : 0;
  q.hi = a <= S ? min(cu[a], N) : N;
  q.off = 0;
  return q;
}

// Tokens of sequence s: none where the boundaries are out of order or of range.
__device__ __forceinline__ void span_of(const int* cu, int T, int N, int s, int& lo, int& hi) {
  if (cu == nullptr) {
    lo = s * T;
    hi = lo + T;
  } else {
    lo = min(max(cu[s], 0), N);
    hi = min(max(cu[s + 1], lo), N);
  }
}

}  // namespace ltc
