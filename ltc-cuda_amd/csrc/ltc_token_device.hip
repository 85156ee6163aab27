// Log probabilities of given tokens, entropy and top alternatives, and
// distillation from a teacher's top logits, for gfx950. Everything that needs the
// whole vocabulary is one pass over a row's logits x with a running maximum m:
//   S0 = sum exp(y),  S1 = sum exp(y) y,   y = (x - m) / tau,
// rescaled when m grows, from which log p_j = y_j - log S0 and the entropy is
// log S0 - S1 / S0. The backward reads the row once more and writes
//   dL/dx_j = (gl (1[j = id] - p_j) - gH p_j (log p_j + H)) / tau
//   dL/dx_j = tau gl (q_j - sum_{k: id_k = j} p_k)          (distillation)
// A row is one workgroup's, or, with few rows, split over several whose partial
// results a second launch joins. Sums and statistics are fp32; x - m is taken
// before the scaling, so large logits lose nothing to it.
#include <hip/hip_runtime.h>

#include "../../include/ltc_capi.h"
#include "ltc_seq_internal.h"

namespace ltc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Start of the running maximum: below every finite logit of the types, and
// finite, so that -inf - m stays -inf.
constexpr float kLowest = -3.402823466e38f;
constexpr int kWaves = kTokThreads / 64;

// Running statistics in powers of two: s0 = sum 2^z, s1 = sum 2^z z, z = (x - m) c.
struct Stat {
  float m, s0, s1;
};
__device__ __forceinline__ Stat no_stat() { return Stat{kLowest, 0.f, 0.f}; }

// z for products with 2^z, which is 0 long before: z itself may be -inf.
__device__ __forceinline__ float finite_z(float z) { return fmaxf(z, -1.0e4f); }

template <bool ENT>
__device__ __forceinline__ void rescale(Stat& s, float m, float c) {
  const float dz = (s.m - m) * c;  // <= 0; -inf where nothing was before
  const float f = __builtin_amdgcn_exp2f(dz);
  if constexpr (ENT) s.s1 = f * fmaf(finite_z(dz), s.s0, s.s1);
  s.s0 *= f;
  s.m = m;
}

template <bool ENT>
__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  rescale<ENT>(a, m, c);
  rescale<ENT>(b, m, c);
  a.s0 += b.s0;
  a.s1 += b.s1;
  return a;
}

// Order of alternatives as one integer: larger logits first (NaN before all),
// equal ones by the lower index. 0 is no entry.
__device__ __forceinline__ unsigned ordered(float x) {
  x += 0.f;  // -0 and +0 are equal
  const unsigned u = __float_as_uint(x);
  if (!(x == x)) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned k) {
  if (k == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ unsigned long long top_key(float x, int j) {
  return (unsigned long long)ordered(x) << 32 | (0xffffffffu - (unsigned)j);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xffffffffu - (unsigned)k); }
__device__ __forceinline__ float key_value(unsigned long long k) { return from_ordered((unsigned)(k >> 32)); }

__device__ __forceinline__ unsigned long long shfl64(unsigned long long v, int src) {
  const unsigned lo = __shfl((unsigned)v, src), hi = __shfl((unsigned)(v >> 32), src);
  return (unsigned long long)hi << 32 | lo;
}

// The best keys a wave has seen, one per lane, descending.
struct TopList {
  unsigned long long key = 0;  // this lane's
  float thr = -__builtin_inff();  // value of the last that counts; -inf: none yet

  __device__ __forceinline__ void insert(unsigned long long k) {
    const int pos = __popcll(__ballot(key > k));
    const int lane = threadIdx.x & 63;
    const unsigned lo = __shfl_up((unsigned)key, 1), hi = __shfl_up((unsigned)(key >> 32), 1);
    const unsigned long long up = (unsigned long long)hi << 32 | lo;
    key = lane < pos ? key : (lane == pos ? k : up);
  }
  // Descending order of the lanes' keys (bitonic).
  __device__ __forceinline__ void sort() {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) {
        const unsigned long long o = shfl64(key, lane ^ j);
        const bool up = (lane & k) != 0, low = (lane & j) == 0;
        const bool take = (low != up) ? o > key : o < key;
        key = take ? o : key;
      }
  }
  __device__ __forceinline__ void set_threshold(int top) {
    const unsigned k = __shfl((unsigned)(key >> 32), top - 1);
    thr = k == 0 ? -__builtin_inff() : from_ordered(k);
  }
};

template <class T, int V>
struct TokVec {
  T v[V];
};

// Best `top` of n keys in LDS (any order, 0: none), written in order by rank.
__device__ __forceinline__ void write_top(const unsigned long long* keys, int n, int top,
                                          unsigned long long* best) {
  for (int i = threadIdx.x; i < n; i += kTokThreads) {
    const unsigned long long k = keys[i];
    if (k == 0) continue;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > k;
    if (rank < top) best[rank] = k;
  }
}

__device__ __forceinline__ long long id_at(const void* ids, int id64, long long i) {
  return id64 ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
}

// Per thread loops over a segment [j0, j1) of a row: the part before the first
// 16-byte boundary and the rest by single logits, in between 16 bytes a thread.
// f(value, index) sees the single ones, fv(vector, first index) the others.
template <class T, class F1, class FV>
__device__ __forceinline__ void each_logit(const T* row, int j0, int j1, F1&& f, FV&& fv) {
  constexpr int V = 16 / (int)sizeof(T);
  const int off = (int)(((16 - ((uintptr_t)(row + j0) & 15)) & 15) / sizeof(T));
  const int a = j0 + off < j1 ? j0 + off : j1;
  const int nv = (j1 - a) / V, b = a + nv * V;
  // the loop's trip count is the same for every thread: f and fv may use the wave
  for (int i = 0; i < nv; i += kTokThreads) {
    const int q = i + threadIdx.x;
    const bool in = q < nv;
    TokVec<T, V> x{};
    if (in) x = *reinterpret_cast<const TokVec<T, V>*>(__builtin_assume_aligned(row + a + (long long)q * V, 16));
    fv(x, a + q * V, in);
  }
  const int head = a - j0, tail = j1 - b;  // below V each
  if (head + tail > 0) {
    const int q = threadIdx.x;
    const bool in = q < head + tail;
    const int j = q < head ? j0 + q : b + (q - head);
    f(in ? (float)row[j] : 0.f, j, in);
  }
}

// What a row's statistics give, by the threads of one workgroup, all of which
// call it with the same s.
template <class T>
__device__ void finish_logprobs(const TokArgs& p, long long row, const Stat& s,
                                const unsigned long long* best) {
  const float ls = kLn2 * __builtin_amdgcn_logf(s.s0);  // log S0
  const float H = ls - kLn2 * (s.s1 / s.s0);
  if (threadIdx.x == 0) {
    const long long id = id_at(p.ids, p.id64, row * p.sid);
    float lp = 0.f, en = 0.f;
    if (id >= p.V) {
      lp = en = __builtin_nanf("");
    } else if (id >= 0) {
      const float x = (float)static_cast<const T*>(p.x)[row * p.sx + id];
      lp = (x - s.m) / p.tau - ls;
      en = H;
    }
    p.logp[row] = lp;
    if (p.ent) p.ent[row] = en;
    if (p.stats) {
      p.stats[row * 3] = s.m;
      p.stats[row * 3 + 1] = ls;
      p.stats[row * 3 + 2] = H;
    }
  }
  if ((int)threadIdx.x < p.top) {
    const unsigned long long k = best[threadIdx.x];
    p.top_logp[row * p.top + threadIdx.x] = (key_value(k) - s.m) / p.tau - ls;
    p.top_ids[row * p.top + threadIdx.x] = key_index(k);
  }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// Over the workgroup, in a fixed order; w holds kWaves floats.
__device__ __forceinline__ float block_max(float v, float* w) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = w[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v = fmaxf(v, w[i]);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* w) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
  __syncthreads();
  v = w[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v += w[i];
  return v;
}

__device__ __forceinline__ float teacher_at(const TokArgs& p, long long row, int k) {
  const long long at = row * p.st + k;
  if (p.t_type == LTC_F32) return static_cast<const float*>(p.t)[at];
  if (p.t_type == LTC_BF16) return (float)static_cast<const __bf16*>(p.t)[at];
  return (float)static_cast<const _Float16*>(p.t)[at];
}

// The teacher's maximum and sum over the entries of a row that are there (n of
// them); bad when an id is V or more or a logit NaN or +inf.
struct Teacher {
  float m, s;
  bool some, bad;
};
__device__ __forceinline__ Teacher teacher_of(const TokArgs& p, long long row, float* w) {
  const float c = p.c;
  float m = -__builtin_inff(), bad = 0.f;
  for (int k = threadIdx.x; k < p.K; k += kTokThreads) {
    const long long id = id_at(p.ids, p.id64, row * p.sid + k);
    if (id >= p.V) bad = 1.f;
    if (id >= 0) {
      const float t = teacher_at(p, row, k);
      m = fmaxf(m, t);
      if (!(t < __builtin_inff())) bad = 1.f;
    }
  }
  Teacher r;
  r.m = block_max(m, w);
  r.bad = block_max(bad, w) > 0.f;
  r.some = r.m > -__builtin_inff();
  float s = 0.f;
  for (int k = threadIdx.x; k < p.K; k += kTokThreads) {
    const long long id = id_at(p.ids, p.id64, row * p.sid + k);
    if (id >= 0 && r.some) s += __builtin_amdgcn_exp2f((teacher_at(p, row, k) - r.m) * c);
  }
  r.s = block_sum(s, w);
  return r;
}

template <class T>
__device__ void finish_distill(const TokArgs& p, long long row, const Stat& s, float* w) {
  const float ls = kLn2 * __builtin_amdgcn_logf(s.s0);
  const Teacher t = teacher_of(p, row, w);
  const float lt = kLn2 * __builtin_amdgcn_logf(t.s);
  float sum = 0.f;
  if (t.some && !t.bad)
    for (int k = threadIdx.x; k < p.K; k += kTokThreads) {
      const long long id = id_at(p.ids, p.id64, row * p.sid + k);
      if (id < 0) continue;
      const float y = (teacher_at(p, row, k) - t.m) / p.tau - lt;
      const float pk = __builtin_amdgcn_exp2f(y * kLog2e);
      const float x = (float)static_cast<const T*>(p.x)[row * p.sx + id];
      if (pk > 0.f) sum += pk * (y - ((x - s.m) / p.tau - ls));
    }
  sum = block_sum(sum, w);
  if (threadIdx.x == 0) {
    p.logp[row] = t.bad ? __builtin_nanf("") : p.tau * p.tau * sum;
    if (p.stats) {
      p.stats[row * 3] = s.m;
      p.stats[row * 3 + 1] = ls;
      p.stats[row * 3 + 2] = 0.f;
    }
  }
}

enum : int { kLogprobs = 0, kDistill = 1 };

// One segment of a row; whole rows are finished here.
template <class T, int OP, bool ENT, bool TOP>
__global__ __launch_bounds__(kTokThreads) void tok_fwd_kernel(TokArgs p) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ Stat ws[kWaves];
  __shared__ float w[kWaves];
  __shared__ unsigned long long keys[TOP ? kWaves * kTopMax : 1], best[TOP ? kTopMax : 1];
  const long long row = blockIdx.x / p.nsplit;
  const int sp = blockIdx.x % p.nsplit;
  const int j0 = sp * p.seg, j1 = j0 + p.seg < p.V ? j0 + p.seg : p.V;
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  const float c = p.c;
  Stat s = no_stat();
  TopList tl;
  bool first = true;

  auto offer = [&](const float(&y)[V], int j, bool in, int nv) {
    // at most one bit per value of this lane
    unsigned cand = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nv && in && !(y[v] < tl.thr)) cand |= 1u << v;
    if (!__any(cand != 0)) return;
    if (first) {
      // the lanes' largest values start the list: almost nothing else passes it
      unsigned long long k = 0;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (cand >> v & 1) {
          const unsigned long long q = top_key(y[v], j + v);
          if (q > k) k = q;
        }
      if (k != 0) cand &= ~(1u << (key_index(k) - j));
      tl.key = k;
      tl.sort();
      tl.set_threshold(p.top);
      first = false;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const unsigned long long k = (cand >> v & 1) && !(y[v] < tl.thr) ? top_key(y[v], j + v) : 0;
      unsigned long long mask = __ballot(k != 0);
      while (mask != 0) {
        const int src = __ffsll((long long)mask) - 1;
        mask &= mask - 1;
        const unsigned long long q = shfl64(k, src);
        if (q > shfl64(tl.key, p.top - 1)) {
          tl.insert(q);
          tl.set_threshold(p.top);
        }
      }
    }
  };
  auto add = [&](const float(&y)[V], int nv) {
    float mx = y[0];
#pragma unroll
    for (int v = 1; v < V; ++v)
      if (v < nv) mx = fmaxf(mx, y[v]);
    if (mx > s.m) rescale<ENT>(s, mx, c);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nv) {
        const float z = (y[v] - s.m) * c;
        const float e = __builtin_amdgcn_exp2f(z);
        s.s0 += e;
        if constexpr (ENT) s.s1 = fmaf(e, finite_z(z), s.s1);
      }
  };
  each_logit(
      x, j0, j1,
      [&](float v, int j, bool in) {
        float y[V] = {v};
        if (in) add(y, 1);
        if constexpr (TOP) offer(y, j, in, 1);
      },
      [&](const TokVec<T, V>& q, int j, bool in) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = (float)q.v[v];
        if (in) add(y, V);
        if constexpr (TOP) offer(y, j, in, V);
      });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor(s.m, o);
    b.s0 = __shfl_xor(s.s0, o);
    b.s1 = __shfl_xor(s.s1, o);
    s = merge<ENT>(s, b, c);
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane == 0) ws[wave] = s;
  if constexpr (TOP)
    if (lane < p.top) keys[wave * p.top + lane] = tl.key;
  __syncthreads();
  s = ws[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) s = merge<ENT>(s, ws[i], c);
  if constexpr (TOP) {
    if ((int)threadIdx.x < p.top) best[threadIdx.x] = 0;
    __syncthreads();
    write_top(keys, kWaves * p.top, p.top, best);
    __syncthreads();
  }
  if (p.nsplit == 1) {
    if constexpr (OP == kLogprobs) finish_logprobs<T>(p, row, s, best);
    else finish_distill<T>(p, row, s, w);
  } else {
    const long long at = row * p.nsplit + sp;
    if (threadIdx.x == 0) {
      p.part[at * 3] = s.m;
      p.part[at * 3 + 1] = s.s0;
      p.part[at * 3 + 2] = s.s1;
    }
    if constexpr (TOP)
      if ((int)threadIdx.x < p.top) p.part_top[at * p.top + threadIdx.x] = best[threadIdx.x];
  }
}

// Rows split over workgroups: joins their parts, in their order.
constexpr int kSplitMax = 64;
template <class T, int OP, bool ENT, bool TOP>
__global__ __launch_bounds__(kTokThreads) void tok_join_kernel(TokArgs p) {
  __shared__ float w[kWaves];
  __shared__ unsigned long long keys[TOP ? kSplitMax * kTopMax : 1], best[TOP ? kTopMax : 1];
  const long long row = blockIdx.x;
  const float c = p.c;
  Stat s = no_stat();
  for (int i = 0; i < p.nsplit; ++i) {
    const float* q = p.part + (row * p.nsplit + i) * 3;
    Stat b;
    b.m = q[0];
    b.s0 = q[1];
    b.s1 = q[2];
    s = merge<ENT>(s, b, c);
  }
  if constexpr (TOP) {
    const int n = p.nsplit * p.top;
    for (int i = threadIdx.x; i < n; i += kTokThreads) keys[i] = p.part_top[row * n + i];
    if ((int)threadIdx.x < p.top) best[threadIdx.x] = 0;
    __syncthreads();
    write_top(keys, n, p.top, best);
    __syncthreads();
  }
  if constexpr (OP == kLogprobs) finish_logprobs<T>(p, row, s, best);
  else finish_distill<T>(p, row, s, w);
}

// One segment of a row's gradient. The few logits that a token or a teacher
// entry names are written again, after the rest.
template <class T, int OP>
__global__ __launch_bounds__(kTokThreads) void tok_bwd_kernel(TokArgs p) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float w[kWaves];
  __shared__ float pk[OP == kDistill ? kTeacherMax : 1];
  __shared__ int ik[OP == kDistill ? kTeacherMax : 1];
  const long long row = blockIdx.x / p.nsplit;
  const int sp = blockIdx.x % p.nsplit;
  const int j0 = sp * p.seg, j1 = j0 + p.seg < p.V ? j0 + p.seg : p.V;
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  T* gx = static_cast<T*>(p.gx) + row * p.V;
  const float c = p.c;
  const float m = p.stats[row * 3], ls = p.stats[row * 3 + 1], H = p.stats[row * 3 + 2];
  // dL/dx_j = p_j (k0 + k1 log2 p_j) + what the named ones add
  float k0, k1 = 0.f, named = 0.f;
  long long id = -1;
  if constexpr (OP == kLogprobs) {
    id = id_at(p.ids, p.id64, row * p.sid);
    float gl = p.gp ? p.gp[row * p.sgp] : 0.f, ge = p.ge ? p.ge[row * p.sge] : 0.f;
    if (id < 0) gl = ge = 0.f;
    if (id >= p.V) gl = __builtin_nanf("");
    named = gl * p.inv_tau;
    k0 = gl == 0.f && ge == 0.f ? 0.f : -(gl + ge * H) * p.inv_tau;
    k1 = -ge * p.inv_tau * kLn2;
  } else {
    const Teacher t = teacher_of(p, row, w);
    const float g = t.bad ? __builtin_nanf("") : (t.some ? p.tau * p.gp[row * p.sgp] : 0.f);
    const float inv = t.some ? 1.f / t.s : 0.f;
    for (int k = threadIdx.x; k < p.K; k += kTokThreads) {
      const long long q = id_at(p.ids, p.id64, row * p.sid + k);
      const bool there = q >= 0 && q < p.V && t.some;
      ik[k] = there ? (int)q : -1;
      pk[k] = there ? __builtin_amdgcn_exp2f((teacher_at(p, row, k) - t.m) * c) * inv : 0.f;
    }
    named = -g;
    k0 = g;
  }
  const float l2 = ls * kLog2e;
  // A row without anything to add is zero whatever its logits are.
  const bool none = k0 == 0.f && k1 == 0.f;
  auto grad = [&](float xj) {
    const float l = fmaf(xj - m, c, -l2);  // log2 p_j
    const float pj = __builtin_amdgcn_exp2f(l);
    if (none) return 0.f;
    if constexpr (OP == kLogprobs) return pj * fmaf(k1, finite_z(l), k0);
    return pj * k0;
  };
  const bool same = (((uintptr_t)(x + j0) ^ (uintptr_t)(gx + j0)) & 15) == 0;
  each_logit(
      x, j0, j1, [&](float v, int j, bool in) { if (in) gx[j] = (T)grad(v); },
      [&](const TokVec<T, V>& q, int j, bool in) {
        if (!in) return;
        TokVec<T, V> o;
#pragma unroll
        for (int v = 0; v < V; ++v) o.v[v] = (T)grad((float)q.v[v]);
        if (same) *reinterpret_cast<TokVec<T, V>*>(__builtin_assume_aligned(gx + j, 16)) = o;
        else __builtin_memcpy(gx + j, &o, sizeof(o));
      });
  __syncthreads();
  if constexpr (OP == kLogprobs) {
    if (threadIdx.x == 0 && id >= j0 && id < j1) gx[id] = (T)(grad((float)x[id]) + named);
  } else {
    for (int k = threadIdx.x; k < p.K; k += kTokThreads) {
      const int j = ik[k];
      if (j < j0 || j >= j1) continue;
      float sum = 0.f;
      for (int q = 0; q < p.K; ++q) sum += ik[q] == j ? pk[q] : 0.f;
      gx[j] = (T)(none ? 0.f : fmaf(named, sum, grad((float)x[j])));
    }
  }
}

template <class F>
hipError_t with_type(int x_type, F&& f) {
  if (x_type == LTC_F32) return f(float{});
  if (x_type == LTC_BF16) return f(__bf16{});
  return f(_Float16{});
}

template <class T, int OP, bool ENT, bool TOP>
hipError_t fwd(const TokArgs& a, hipStream_t s) {
  LTC_LAUNCH((tok_fwd_kernel<T, OP, ENT, TOP>), dim3((unsigned)(a.N * a.nsplit)), dim3(kTokThreads), 0,
             s, a);
  if (a.nsplit > 1)
    LTC_LAUNCH((tok_join_kernel<T, OP, ENT, TOP>), dim3((unsigned)a.N), dim3(kTokThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

void tok_split(long long N, int V, int elem_bytes, int* nsplit, int* seg) {
  // whole rows keep 1024 workgroups busy; fewer are cut, to no less than four
  // 16-byte loads of every thread
  const int vec = 16 / elem_bytes, least = 4 * kTokThreads * vec;
  long long n = N < 1 || N >= 1024 ? 1 : (1024 + N - 1) / N;
  if (n > (V + least - 1) / least) n = (V + least - 1) / least;
  if (n > kSplitMax) n = kSplitMax;
  if (n < 1) n = 1;
  long long sg = (V + n - 1) / n;
  sg = (sg + vec - 1) / vec * vec;
  *seg = (int)sg;
  *nsplit = (int)((V + sg - 1) / sg);
}

hipError_t launch_logprobs_fwd(int x_type, const TokArgs& a, hipStream_t s) {
  return with_type(x_type, [&](auto t) {
    using T = decltype(t);
    return a.top > 0 ? fwd<T, kLogprobs, true, true>(a, s) : fwd<T, kLogprobs, true, false>(a, s);
  });
}

hipError_t launch_distill_fwd(int x_type, const TokArgs& a, hipStream_t s) {
  return with_type(x_type, [&](auto t) { return fwd<decltype(t), kDistill, false, false>(a, s); });
}

template <int OP>
static hipError_t bwd(int x_type, const TokArgs& a, hipStream_t s) {
  return with_type(x_type, [&](auto t) {
    LTC_LAUNCH((tok_bwd_kernel<decltype(t), OP>), dim3((unsigned)(a.N * a.nsplit)), dim3(kTokThreads),
               0, s, a);
    return hipGetLastError();
  });
}

hipError_t launch_logprobs_bwd(int x_type, const TokArgs& a, hipStream_t s) {
  return bwd<kLogprobs>(x_type, a, s);
}
hipError_t launch_distill_bwd(int x_type, const TokArgs& a, hipStream_t s) {
  return bwd<kDistill>(x_type, a, s);
}

}  // namespace ltc
