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

#include <type_traits>

#include "../../include/ltc_capi.h"
#include "ltc_seq_internal.h"
#include "ltc_vec.h"

namespace ltc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Start of the running maximum: below every finite logit of the types, and
// finite, so that -inf - m stays -inf.
constexpr float kLowest = -3.402823466e38f;
constexpr int kWaves = kTokThreads / 64;

// Running statistics in powers of two: s0 = sum 2^z, s1 = sum 2^z z, z = (x - m) c,
// c = log2(e) / tau. The difference is taken first: a row of the type's lowest value
// alone (a mask that leaves nothing) is then uniform, as it is by the definition.
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

// Of all lanes, in every lane.
template <bool ENT>
__device__ __forceinline__ Stat merge_wave(Stat s, float c) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor(s.m, o);
    b.s0 = __shfl_xor(s.s0, o);
    b.s1 = __shfl_xor(s.s1, o);
    s = merge<ENT>(s, b, c);
  }
  return s;
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

__device__ __forceinline__ unsigned long long lane64(unsigned long long v, int src) {
  const unsigned lo = __builtin_amdgcn_readlane((unsigned)v, src);
  const unsigned hi = __builtin_amdgcn_readlane((unsigned)(v >> 32), src);
  return (unsigned long long)hi << 32 | lo;
}
// The lane before's value; 0 in the first.
__device__ __forceinline__ unsigned from_left(unsigned v) {
  return __builtin_amdgcn_update_dpp(0u, v, 0x138 /* wave_shr:1 */, 0xf, 0xf, false);
}

// The best keys a wave has seen, one per lane, descending: whatever the logits are,
// it holds them.
struct TopList {
  unsigned long long key;   // this lane's; 0: none
  unsigned long long last;  // the last that counts
  float thr;                // its value; -inf: none yet

  __device__ __forceinline__ void clear() {
    key = last = 0;
    thr = -__builtin_inff();
  }
  __device__ __forceinline__ void insert(unsigned long long k) {
    const int pos = __popcll(__ballot(key > k));
    const int lane = threadIdx.x & 63;
    const unsigned long long up =
        (unsigned long long)from_left((unsigned)(key >> 32)) << 32 | from_left((unsigned)key);
    key = lane < pos ? key : (lane == pos ? k : up);
  }
  __device__ __forceinline__ void set_threshold(int top) {
    last = lane64(key, top - 1);
    thr = last == 0 ? -__builtin_inff() : key_value(last);
  }
};

// Best `top` of n keys in LDS (any order, 0: none), written in order by rank.
__device__ __forceinline__ void write_top(const unsigned long long* keys, int n, int top,
                                          unsigned long long* best) {
  for (int i = threadIdx.x; i < n; i += kTokThreads) {
    const unsigned long long k = keys[i];
    if (k == 0) continue;
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += keys[j] > k;
    if (rank < top) best[rank] = k;
  }
}

__device__ __forceinline__ long long id_at(const void* ids, int id64, long long i) {
  return id64 ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
}

// A workgroup's walk over a segment [j0, j1) of a row: the part before the first
// 16-byte boundary and the rest by single logits, in between 16 bytes a thread,
// UNROLL loads of each thread under way at once. f(value, index, there) sees the
// single ones, fv(vector, first index, there) the others; every thread of the
// workgroup comes by the same number of times, so they may use the wave.
template <int UNROLL, class T, class F1, class FV>
__device__ __forceinline__ void each_logit(const T* row, int j0, int j1, F1&& f, FV&& fv) {
  constexpr int V = 16 / (int)sizeof(T);
  const int off = (int)(((16 - ((uintptr_t)(row + j0) & 15)) & 15) / sizeof(T));
  const int a = j0 + off < j1 ? j0 + off : j1;
  const int nv = (j1 - a) / V, b = a + nv * V;
  const T* base = row + a;
  auto load = [&](int q) {
    Vec<T, V> r;
    __builtin_memcpy(r.w, __builtin_assume_aligned(base + (long long)q * V, 16), 16);
    return r;
  };
  int i = 0;
  for (; i + UNROLL * kTokThreads <= nv; i += UNROLL * kTokThreads) {
    Vec<T, V> x[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) x[u] = load(i + u * kTokThreads + threadIdx.x);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) fv(x[u], a + (i + u * kTokThreads + (int)threadIdx.x) * V, true);
  }
  for (; i < nv; i += kTokThreads) {
    const int q = i + threadIdx.x;
    const bool in = q < nv;
    Vec<T, V> x{};
    if (in) x = load(q);
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

// The best of a segment, collected on the walk that forms its statistics. Every
// thread's largest logit so far is at hand (its running maximum), and the best of a
// workgroup's are bounded from below by
//   the least over the waves of each wave's (top / 4)-th largest lane maximum, and
//   any wave's top-th largest lane maximum,
// since as many logits reach them. What does not reach the bound is out; what does
// goes to a list, of which the best are taken by rank at the end. The bound is
// formed again after 1, 2, 4, ... vectors of a thread; 100 to 200 entries come
// together. If more than kCollect come together
// (ties; rising logits; masks that leave little else), a second walk keeps ordered
// lists instead, which hold whatever the logits are.
constexpr int kCollect = 512;
struct TopShared {
  unsigned long long keys[kCollect], kept[kCollect], best[kTopMax];
  float bound[kWaves], own[kWaves];
  int n, nkept;
};
struct NoTop {};

// The largest of the wave's values (as ordered() numbers them), its lane's set to 0.
__device__ __forceinline__ unsigned take_max(unsigned& v) {
  unsigned m = v;
  // over rows of 16 lanes, then across them: the last lane has seen all
#define LTC_DPP_MAX(ctrl)                                                                   \
  {                                                                                         \
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, ctrl, 0xf, 0xf, false); \
    m = m > o ? m : o;                                                                      \
  }
  LTC_DPP_MAX(0x111)  // row_shr:1
  LTC_DPP_MAX(0x112)
  LTC_DPP_MAX(0x114)
  LTC_DPP_MAX(0x118)
  LTC_DPP_MAX(0x142)  // row_bcast:15
  LTC_DPP_MAX(0x143)  // row_bcast:31
#undef LTC_DPP_MAX
  m = (unsigned)__builtin_amdgcn_readlane((int)m, 63);
  const unsigned long long at = __ballot(v == m);
  if ((threadIdx.x & 63) == (unsigned)(__ffsll((long long)at) - 1)) v = 0;
  return m;
}

struct Collect {
  TopShared& sh;
  int top;
  bool full;  // every thread of the workgroup has a vector, more than one
  float bound = -__builtin_inff();
  int vectors = 0;                              // of each thread
  int next = 1;                                 // when the bound is formed again

  __device__ __forceinline__ Collect(TopShared& s, int t, bool f) : sh(s), top(t), full(f) {
    if (threadIdx.x == 0) sh.n = sh.nkept = 0;
    if ((int)threadIdx.x < t) sh.best[threadIdx.x] = 0;
    if (threadIdx.x < kWaves) sh.bound[threadIdx.x] = sh.own[threadIdx.x] = -__builtin_inff();
    __syncthreads();
  }
  // The waves' bounds as they are now. They only rise: one read late is lower, and
  // holds as well.
  __device__ __forceinline__ void reread() {
    asm volatile("" ::: "memory");
    float low = sh.bound[0], k = sh.own[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
      low = fminf(low, sh.bound[i]);
      k = fmaxf(k, sh.own[i]);
    }
    bound = fmaxf(bound, fmaxf(low, k));
  }
  // largest: this thread's largest logit so far, or kLowest. All waves come by
  // together the first time and at the end.
  __device__ __forceinline__ void raise(float largest, bool end) {
    const int quarter = (top + kWaves - 1) / kWaves, wave = threadIdx.x >> 6;
    // a wave without logits would hold the least of the waves down for good
    const bool begin = next == 1;
    const int n = begin && !full ? top : quarter;
    next *= 2;
    // a thread that has seen nothing over the lowest bounds nothing
    unsigned q = ordered(largest == kLowest ? -__builtin_inff() : largest), m = 0;
    for (int i = 0; i < n; ++i) {
      m = take_max(q);
      if (i == quarter - 1 && (threadIdx.x & 63) == 0) sh.bound[wave] = from_ordered(m);
    }
    if (n == top && (threadIdx.x & 63) == 0) sh.own[wave] = from_ordered(m);
    if (begin || end) __syncthreads();
    reread();
  }
  // Takes in one value a lane (key 0: none).
  __device__ __forceinline__ void take(unsigned long long k) {
    const int lane = threadIdx.x & 63;
    const unsigned long long mask = __ballot(k != 0);
    int base = 0;
    if (lane == 0) base = atomicAdd(&sh.n, (int)__popcll(mask));
    base = __builtin_amdgcn_readfirstlane(base);
    const int at = base + (int)__popcll(mask & ((1ull << lane) - 1));
    if (k != 0 && at < kCollect) sh.keys[at] = k;
  }
  template <class T, int V>
  __device__ __forceinline__ void offer(const Vec<T, V>& q, float largest, float so_far, int j, bool in) {
    if (++vectors == next) raise(so_far, false);
    if (!__any(in && !(largest < bound))) return;
    reread();
    if (!__any(in && !(largest < bound))) return;
    unsigned cand = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) cand |= !(q.get(v) < bound) ? 1u << v : 0u;
    if (!in) cand = 0;
    while (__any(cand != 0)) {
      const int at = (__ffs((int)cand) - 1) & (V - 1);
      take(cand != 0 ? top_key(q.get_at(at), j + at) : 0ull);
      cand &= cand - 1;
    }
  }
  __device__ __forceinline__ void offer(float y, int j, bool in) {
    const bool reaches = in && !(y < bound);
    if (__any(reaches)) take(reaches ? top_key(y, j) : 0ull);
  }
  // The best, in sh.best (0 where there are none) after the next barrier.
  template <class T>
  __device__ __forceinline__ void finish(const T* x, int j0, int j1, float largest) {
    constexpr int V = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    raise(largest, true);  // with a barrier: all entries are in, too
    int n = sh.n;
    if (n <= kCollect) {
      // most entries came in under a lower bound
      for (int i = threadIdx.x; i < n; i += kTokThreads) {
        const unsigned long long k = sh.keys[i];
        if (!(key_value(k) < bound)) sh.kept[atomicAdd(&sh.nkept, 1)] = k;
      }
      __syncthreads();
      n = sh.nkept;
    } else {
      TopList tl;
      tl.clear();
      auto add = [&](unsigned long long k) {
        unsigned long long mask = __ballot(k > tl.last);
        while (mask != 0) {
          const int src = __ffsll((long long)mask) - 1;
          mask &= mask - 1;
          const unsigned long long q = lane64(k, src);
          if (q > tl.last) {
            tl.insert(q);
            tl.set_threshold(top);
          }
        }
      };
      each_logit<4>(
          x, j0, j1, [&](float y, int j, bool in) { add(in ? top_key(y, j) : 0ull); },
          [&](const Vec<T, V>& q, int j, bool in) {
            bool any = false;
#pragma unroll
            for (int v = 0; v < V; ++v) any = any || !(q.get(v) < tl.thr);
            if (!__any(in && any)) return;
#pragma unroll
            for (int v = 0; v < V; ++v) add(in ? top_key(q.get(v), j + v) : 0ull);
          });
      __syncthreads();
      if (lane < top) sh.kept[wave * top + lane] = tl.key;
      n = kWaves * top;
      __syncthreads();
    }
    write_top(sh.kept, n, top, sh.best);
  }
};

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
    p.top_ids[row * p.top + threadIdx.x] = k == 0 ? 0 : key_index(k);  // 0: a row of NaN
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
      p.stats[row * 4] = s.m;
      p.stats[row * 4 + 1] = ls;
      // NaN: no loss; -inf: no entries
      p.stats[row * 4 + 2] = t.bad ? __builtin_nanf("") : t.m;
      p.stats[row * 4 + 3] = lt;
    }
  }
}

enum : int { kLogprobs = 0, kDistill = 1 };

// One segment of a row; whole rows are finished here. Long rows are bound by their
// bytes, and 16-bit ones as much by arithmetic, about 11 instructions a logit with the
// entropy: 2047 rows of 50021 fp32 with the best 5 78 us, 5.2 TB/s; 4096 rows of 32768
// bf16 45 us alone, 5.9 TB/s, and 76 with the best 20.
template <class T, int OP, bool ENT, bool TOP>
__global__ __launch_bounds__(kTokThreads) void tok_fwd_kernel(TokArgs p) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ Stat ws[kWaves];
  __shared__ float w[kWaves];
  __shared__ typename std::conditional<TOP, TopShared, NoTop>::type tops;
  const long long row = blockIdx.x / p.nsplit;
  const int sp = blockIdx.x % p.nsplit;
  const int j0 = sp * p.seg, j1 = j0 + p.seg < p.V ? j0 + p.seg : p.V;
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  const float c = p.c;
  Stat s = no_stat();
  // takes nv values in; the largest of them
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
    return mx;
  };
  auto walk = [&](auto&& one, auto&& many) {
    each_logit<4>(
        x, j0, j1,
        [&](float v, int j, bool in) {
          const float y[V] = {v};
          if (in) add(y, 1);
          one(v, j, in);
        },
        [&](const Vec<T, V>& q, int j, bool in) {
          float y[V], mx = 0.f;
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] = q.get(v);
          if (in) mx = add(y, V);
          many(q, mx, j, in);
        });
  };
  if constexpr (TOP) {
    Collect best(tops, p.top, j1 - j0 >= 2 * V * kTokThreads);
    walk([&](float v, int j, bool in) { best.offer(v, j, in); },
         [&](const Vec<T, V>& q, float mx, int j, bool in) { best.offer(q, mx, s.m, j, in); });
    best.finish(x, j0, j1, s.m);
  } else {
    walk([](float, int, bool) {}, [](const Vec<T, V>&, float, int, bool) {});
  }
  s = merge_wave<ENT>(s, c);
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
  __syncthreads();
  s = ws[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) s = merge<ENT>(s, ws[i], c);
  const unsigned long long* best = nullptr;
  if constexpr (TOP) best = tops.best;
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

// Rows split over workgroups: joins their parts, a lane of each wave to a part.
constexpr int kSplitMax = 64, kJoinKeys = 512;
static_assert(kJoinKeys >= kTopMax && kCollect >= kWaves * kTopMax, "one list at least");
template <class T, int OP, bool ENT, bool TOP>
__global__ __launch_bounds__(kTokThreads) void tok_join_kernel(TokArgs p) {
  __shared__ float w[kWaves];
  __shared__ unsigned long long keys[TOP ? kJoinKeys : 1], kept[TOP ? kJoinKeys : 1], best[TOP ? kTopMax : 1];
  __shared__ int nkept;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  Stat s = no_stat();
  if (lane < p.nsplit) {
    const float* q = p.part + (row * p.nsplit + lane) * 3;
    s.m = q[0];
    s.s0 = q[1];
    s.s1 = q[2];
  }
  if constexpr (TOP) {
    const int n = p.nsplit * p.top;
    for (int i = threadIdx.x; i < n; i += kTokThreads) keys[i] = p.part_top[row * n + i];
    if ((int)threadIdx.x < p.top) best[threadIdx.x] = 0;
    if (threadIdx.x == 0) nkept = 0;
    __syncthreads();
    // The parts' lists are in order. As many keys as are wanted reach the least of
    // their (top / parts)-th, and the last of any (by rank over all 500 keys of 25
    // parts this took 19 us).
    const int share = (p.top + p.nsplit - 1) / p.nsplit;
    unsigned long long low = ~0ull, bound = 0;
#pragma unroll 8
    for (int i = 0; i < p.nsplit; ++i) {
      const unsigned long long k = keys[i * p.top + share - 1], l = keys[(i + 1) * p.top - 1];
      low = k < low ? k : low;
      bound = l > bound ? l : bound;
    }
    bound = low > bound ? low : bound;
    for (int i = threadIdx.x; i < n; i += kTokThreads) {
      const unsigned long long k = keys[i];
      if (k >= bound && k != 0) kept[atomicAdd(&nkept, 1)] = k;
    }
    __syncthreads();
    write_top(kept, nkept, p.top, best);
    __syncthreads();
  }
  s = merge_wave<ENT>(s, p.c);
  if constexpr (OP == kLogprobs) finish_logprobs<T>(p, row, s, best);
  else finish_distill<T>(p, row, s, w);
}

// One segment of a row's gradient. The few logits that a token or a teacher
// entry names are written again, after the rest. Bound by its bytes, the row read and
// written.
template <class T, int OP>
__global__ __launch_bounds__(kTokThreads) void tok_bwd_kernel(TokArgs p) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float pk[OP == kDistill ? kTeacherMax : 1];
  __shared__ int ik[OP == kDistill ? kTeacherMax : 1];
  __shared__ int count[OP == kDistill ? kTeacherMax / 64 : 1];
  const long long row = blockIdx.x / p.nsplit;
  const int sp = blockIdx.x % p.nsplit;
  const int j0 = sp * p.seg, j1 = j0 + p.seg < p.V ? j0 + p.seg : p.V;
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  T* gx = static_cast<T*>(p.gx) + row * p.V;
  const float c = p.c;
  const float* st = p.stats + row * (OP == kDistill ? 4 : 3);
  const float m = st[0], ls = st[1];
  // the row's entries are under way while it is walked
  constexpr int kEntries = OP == kDistill ? kTeacherMax / kTokThreads : 1;
  long long tid[kEntries];
  float tl[kEntries];
  if constexpr (OP == kDistill) {
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int k = threadIdx.x + i * kTokThreads;
      tid[i] = -1;
      tl[i] = 0.f;
      if (k < p.K) {
        tid[i] = id_at(p.ids, p.id64, row * p.sid + k);
        tl[i] = teacher_at(p, row, k);
      }
    }
  }
  // dL/dx_j = p_j (k0 + k1 log2 p_j) + what the named ones add
  float k0, k1 = 0.f, named = 0.f;
  long long id = -1;
  if constexpr (OP == kLogprobs) {
    id = id_at(p.ids, p.id64, row * p.sid);
    float gl = p.gp ? p.gp[row * p.sgp] : 0.f, ge = p.ge ? p.ge[row * p.sge] : 0.f;
    if (id < 0) gl = ge = 0.f;
    if (id >= p.V) gl = __builtin_nanf("");
    named = gl * p.inv_tau;
    k0 = gl == 0.f && ge == 0.f ? 0.f : -(gl + ge * st[2]) * p.inv_tau;
    k1 = -ge * p.inv_tau * kLn2;
  } else {
    const float tm = st[2];
    const float g = tm == -__builtin_inff() ? 0.f : tm == tm ? p.tau * p.gp[row * p.sgp] : tm;
    named = -g;
    k0 = g;
  }
  if (k0 == 0.f && k1 == 0.f) {
    // a row without anything to add is zero whatever its logits are
    for (int j = j0 + threadIdx.x; j < j1; j += kTokThreads) gx[j] = (T)0.f;
    return;
  }
  const float l2 = ls * kLog2e;
  auto grad = [&](float xj) {
    const float l = fmaf(xj - m, c, -l2);  // log2 p_j
    const float pj = __builtin_amdgcn_exp2f(l);
    if constexpr (OP == kLogprobs) return pj * fmaf(k1, finite_z(l), k0);
    return pj * k0;
  };
  each_logit<4>(
      x, j0, j1, [&](float v, int j, bool in) { if (in) gx[j] = (T)grad(v); },
      [&](const Vec<T, V>& q, int j, bool in) {
        if (!in) return;
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = grad(q.get(v));
        Vec<T, V> r;
        r.put(o);
        store_vec<T, V>(gx + j, r, V);
      });
  if constexpr (OP == kLogprobs) {
    __syncthreads();
    if (threadIdx.x == 0 && id >= j0 && id < j1) gx[id] = (T)(grad((float)x[id]) + named);
  } else {
    // The segment's entries, in their order: each looks through those of the segment
    // for its like, not through all (4096 rows of 65536, K 1024: 290 us and 667).
    const float tm = st[2], lt = st[3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned long long here[kEntries];
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      here[i] = __ballot(tid[i] >= j0 && tid[i] < j1);
      if (lane == 0) count[i * kWaves + wave] = (int)__popcll(here[i]);
    }
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int i = 0; i < kEntries; ++i)
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w == wave && (here[i] >> lane & 1)) {
          const int at = n + (int)__popcll(here[i] & ((1ull << lane) - 1));
          ik[at] = (int)tid[i];
          pk[at] = __builtin_amdgcn_exp2f(((tl[i] - tm) / p.tau - lt) * kLog2e);
        }
        n += count[i * kWaves + w];
      }
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += kTokThreads) {
      const int j = ik[k];
      const float xj = (float)x[j];
      float sum = 0.f;
#pragma unroll 8
      for (int q = 0; q < n; ++q) sum += ik[q] == j ? pk[q] : 0.f;
      gx[j] = (T)fmaf(named, sum, grad(xj));
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

void tok_split(long long N, int V, int elem_bytes, int top, int* nsplit, int* seg) {
  // 1024 rows fill the chip; fewer are cut, to no less than one load of every thread
  // (8 rows of 32000 bf16: 6.3 us in both launches with one, 6.9 with four; top 20
  // 14.2 and 15.1), and to what the join orders at once.
  const int vec = 16 / elem_bytes, least = kTokThreads * vec;
  long long n = N < 1 || N >= 1024 ? 1 : (1024 + N - 1) / N;
  if (n > (V + least - 1) / least) n = (V + least - 1) / least;
  if (n > kSplitMax) n = kSplitMax;
  if (top > 0 && n > kJoinKeys / top) n = kJoinKeys / top;
  if (n < 1) n = 1;
  long long sg = (V + n - 1) / n;
  sg = (sg + vec - 1) / vec * vec;
  *seg = (int)sg;
  *nsplit = (int)((V + sg - 1) / sg);
}

void tok_split_bwd(long long N, int V, int elem_bytes, long long most, int* nsplit, int* seg) {
  // 8 KiB each, so that the chip sweeps through memory and a segment's entries find it
  // still in the L2: 4096 rows of 65536 bf16 176 us (6.1 TB/s), with 16 KiB 183, with
  // 4 KiB 202, with whole rows 209 and, where rows do not align (V 65000), 228.
  constexpr int kBytes = 8192;
  tok_split(N, V, elem_bytes, 0, nsplit, seg);
  const int sg = kBytes / elem_bytes;
  const long long n = ((long long)V + sg - 1) / sg;
  if (sg < *seg && n <= most / N) {
    *seg = sg;
    *nsplit = (int)n;
  }
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
