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

// Which of a batch's L tokens begin a sequence, end one, and lie in one.
template <int L>
struct EdgesOf {
  unsigned start, end, valid;
  // Of the batch at t, up to c1; q is the sequence that was met last.
  __device__ __forceinline__ void find(const int* cu, int S, int T, int N, int t, int c1, Seq& q) {
    start = end = valid = 0;
    const int n = c1 - t < L ? c1 - t : L;
    int i = 0;
    while (i < n) {
      if (t + i < q.lo || t + i >= q.hi) q = seq_of(cu, S, T, N, t + i, 0, 0);
      const int m = q.hi - t < n ? q.hi - t : n;
      if (q.s >= 0) {
        if (q.lo == t + i) start |= 1u << i;
        if (q.hi - t <= n) end |= 1u << (q.hi - t - 1);
        valid |= ((1u << m) - 1) & ~((1u << i) - 1);
      }
      i = m;
    }
  }
  // The tokens of the last sequence in `rest`, which holds valid tokens.
  __device__ __forceinline__ unsigned last(unsigned rest) const {
    const unsigned upto = (2u << (31 - __builtin_clz(rest))) - 1;
    const unsigned begins = upto & start, gaps = upto & ~valid;
    const unsigned lo = begins != 0 ? 1u << (31 - __builtin_clz(begins)) : 0u;
    const unsigned gap = gaps != 0 ? 2u << (31 - __builtin_clz(gaps)) : 0u;
    const unsigned from = lo > gap ? lo : gap;
    return from == 0 ? upto : upto & ~(from - 1);
  }
};

// Calls f with the sequence that token t begins or ends. An edge may have been found by the
// search of another of its sequence's tokens; where boundaries are out of order the search
// of t can end elsewhere, also outside all sequences. Then there is no state, and no call.
template <class F>
__device__ __forceinline__ void at_edge(const int* cu, int S, int T, int N, int t, F&& f) {
  const int s = seq_of(cu, S, T, N, t, 0, 0).s;
  if (s >= 0) f(s);
}

}  // namespace ltc
