// Gated linear recurrence h_t = a_t h_{t-1} + u_t per channel, for gfx950:
//   blend: a = sigmoid(g), u = (1 - a) x      decay: a = exp(g), u = x
// Its backward, with d_t = dL/dh_t + a_{t+1} d_{t+1}:
//   blend: dL/dx = (1 - a) d, dL/dg = d (h_{t-1} - x) a (1 - a)
//   decay: dL/dx = d,         dL/dg = d h_{t-1} a
//
// A run of tokens maps the state that enters it affinely, h -> A h + B, and two
// runs compose to (A2 A1, A2 B1 + B2), so time is cut into tiles: each tile's
// map, then what enters every tile, then every tile's tokens. The tokens of all
// sequences lie end to end; a sequence's first token gives a h0 + u whatever comes
// from before. Decays are never negative, so a map whose A has the sign bit set
// stands for one that drops what enters it, NaN and infinities too. All maps and states are fp32; out and the
// gradients are rounded to their type once, when they are stored.
#include <hip/hip_runtime.h>

#include "../../include/ltc_capi.h"
#include "ltc_seq_internal.h"

namespace ltc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Marks of packed tokens: -1 behind the last sequence (and before the first),
// else 4 * sequence + 1 for its first token + 2 for its last.
constexpr int kMarkNone = -1, kMarkStart = 1, kMarkEnd = 2;

template <class T, int V>
struct Vec {
  T v[V];
};

// n (< V: the row's last channels) of V values at p, which has T's alignment
// only: gfx950 takes wide global loads and stores at any address.
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p, int n) {
  Vec<T, V> r;
  if (n >= V) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) r.v[v] = v < n ? p[v] : T(0.f);
  }
  return r;
}

template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& r, int n) {
  if (n >= V) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < n) p[v] = r.v[v];
  }
}

// a and 1 - a (decay: 1), each to its own relative precision: sigmoid from
// exp(-|g|), which does not overflow. A NaN a has no sign either.
template <int FORM>
__device__ __forceinline__ void gate_of(float g, float& a, float& na) {
  if constexpr (FORM == LTC_GATE_BLEND) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(g) * kLog2e);
    const float r = __builtin_amdgcn_rcpf(1.f + e);
    const float lo = e * r;
    a = fabsf(g < 0.f ? lo : r);
    na = g < 0.f ? r : lo;
  } else {
    a = fabsf(__builtin_amdgcn_exp2f(g * kLog2e));
    na = 1.f;
  }
}

// Where a thread's tokens lie and what they are: bit i of the masks is token i.
template <int LT>
struct Tokens {
  long long t0;           // first token
  unsigned valid, start, end;
  int b[LT];              // sequence of token i
  int r[LT];              // uniform batches: step of token i in its sequence
};

template <int LT, bool PACKED>
__device__ __forceinline__ Tokens<LT> tokens_of(const ScanArgs& p, long long t0) {
  Tokens<LT> k;
  k.t0 = t0;
  k.valid = k.start = k.end = 0;
  int b = 0, r = 0;
  if constexpr (!PACKED) {
    b = (int)(t0 / p.T);
    r = (int)(t0 - (long long)b * p.T);
  }
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    const bool in = t0 + i < p.N;
    if constexpr (PACKED) {
      const int m = in ? p.marks[t0 + i] : kMarkNone;
      k.b[i] = m >> 2;
      k.r[i] = 0;
      if (m >= 0) {
        k.valid |= 1u << i;
        if (m & kMarkStart) k.start |= 1u << i;
        if (m & kMarkEnd) k.end |= 1u << i;
      }
    } else {
      k.b[i] = b;
      k.r[i] = r;
      if (in) {
        k.valid |= 1u << i;
        if (r == 0) k.start |= 1u << i;
        if (r == p.T - 1) k.end |= 1u << i;
      }
      if (++r == p.T) {
        r = 0;
        ++b;
      }
    }
  }
  return k;
}

// Element offset of token i's row.
template <bool PACKED, int LT>
__device__ __forceinline__ long long row_of(const Tokens<LT>& k, int i, long long sb, long long st) {
  if constexpr (PACKED) return (k.t0 + i) * st;
  else return k.b[i] * sb + k.r[i] * st;
}

// A thread's tokens, loaded.
template <class T, class G, int V, int LT>
struct Loaded {
  Vec<T, V> x[LT];
  Vec<G, V> g[LT];
};

template <class T, class G, int V, int LT, bool PACKED>
__device__ __forceinline__ void load_tokens(const ScanArgs& p, const Tokens<LT>& k, int ch, int n,
                                            Loaded<T, G, V, LT>& d) {
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    if (n > 0 && (k.valid >> i & 1)) {
      d.x[i] = load_vec<T, V>(static_cast<const T*>(p.x) + row_of<PACKED>(k, i, p.sxb, p.sxt) + ch, n);
      d.g[i] = load_vec<G, V>(static_cast<const G*>(p.g) + row_of<PACKED>(k, i, p.sgb, p.sgt) + ch, n);
    } else {
      d.x[i] = Vec<T, V>{};
      d.g[i] = Vec<G, V>{};
    }
  }
}

// Initial state of token i's sequence.
template <int V, int LT>
__device__ __forceinline__ Vec<float, V> state_of(const ScanArgs& p, const Tokens<LT>& k, int i, int ch,
                                                  int n) {
  if (p.h0 == nullptr || n <= 0) return Vec<float, V>{};
  return load_vec<float, V>(p.h0 + (long long)k.b[i] * p.H + ch, n);
}

// Whether a map drops what enters it, and what leaves one, h having entered.
__device__ __forceinline__ bool drops(float A) { return __float_as_int(A) < 0; }
__device__ __forceinline__ float leave(float A, float B, float h) { return drops(A) ? B : fmaf(A, h, B); }

// Token i's map (a, u) of every channel; a sequence's first token takes its
// initial state in and drops what comes from before (a = -1), as does a token
// outside all sequences, which gives 0.
template <int FORM, class T, class G, int V, int LT>
__device__ __forceinline__ void maps_of(const ScanArgs& p, const Tokens<LT>& k,
                                        const Loaded<T, G, V, LT>& d, int i, int ch, int n,
                                        float (&a)[V], float (&u)[V]) {
  const bool valid = k.valid >> i & 1;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float na;
    gate_of<FORM>((float)d.g[i].v[v], a[v], na);
    u[v] = na * (float)d.x[i].v[v];
    if (!valid) {
      a[v] = -1.f;
      u[v] = 0.f;
    }
  }
  if (k.start >> i & 1) {
    const Vec<float, V> h0 = state_of<V>(p, k, i, ch, n);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      u[v] = fmaf(a[v], h0.v[v], u[v]);
      a[v] = -1.f;
    }
  }
}

// A workgroup's exchange of its slots' maps: each slot leaves the map of its
// tokens, and every slot gets the map of all slots before it.
template <int CB>
struct SlotMaps {
  static constexpr int kParts = kScanThreads / CB;  // threads per channel
  static constexpr int kPer = kScanSlots / kParts;  // slots per thread
  static_assert(kParts * CB == kScanThreads && kPer * kParts == kScanSlots, "slot split");
  float a[kScanSlots][CB], b[kScanSlots][CB];
  float pa[kParts][CB], pb[kParts][CB];

  template <int V>
  __device__ __forceinline__ void put(int slot, int c, const float (&A)[V], const float (&B)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[slot][c * V + v] = A[v];
      b[slot][c * V + v] = B[v];
    }
  }
  // After a barrier: each slot's map is replaced by that of the slots before it
  // in its part, and the parts' maps are left in pa, pb. Ends without a barrier.
  __device__ __forceinline__ void compose() {
    const int c = threadIdx.x % CB, part = threadIdx.x / CB;
    float A = 1.f, B = 0.f;
#pragma unroll
    for (int s = 0; s < kPer; ++s) {
      const float sa = a[part * kPer + s][c], sb = b[part * kPer + s][c];
      a[part * kPer + s][c] = A;
      b[part * kPer + s][c] = B;
      B = leave(sa, sb, B);
      A = drops(sa) ? sa : A * sa;
    }
    pa[part][c] = A;
    pb[part][c] = B;
  }
  // After another barrier: the whole tile's map of channel c.
  __device__ __forceinline__ void whole(int c, float& A, float& B) {
    A = 1.f;
    B = 0.f;
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      B = leave(pa[q][c], pb[q][c], B);
      A = drops(pa[q][c]) ? pa[q][c] : A * pa[q][c];
    }
  }
  // What enters the slot, from what enters the tile.
  __device__ __forceinline__ float enter(int slot, int c, float h) {
    const int part = slot / kPer;
#pragma unroll
    for (int q = 0; q < kParts; ++q)
      if (q < part) h = leave(pa[q][c], pb[q][c], h);
    return leave(a[slot][c], b[slot][c], h);
  }
};

template <class T>
constexpr int vec_of() {
  return 16 / (int)sizeof(T);
}

// Forward. PHASE 0 leaves each tile's map; PHASE 1 reads what enters each tile
// and runs its tokens.
template <class T, class G, int FORM, bool PACKED, int PHASE>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(ScanArgs p, int cblocks) {
  constexpr int V = vec_of<T>(), CB = kScanLanes * V, LT = kScanTokensFwd;
  __shared__ SlotMaps<CB> sm;
  const int c = threadIdx.x % kScanLanes, slot = threadIdx.x / kScanLanes;
  const long long tile = blockIdx.x / cblocks;
  const int cb = blockIdx.x % cblocks;
  const int ch = cb * CB + c * V;
  const int n = p.H - ch;
  const Tokens<LT> k = tokens_of<LT, PACKED>(p, tile * kScanTileFwd + (long long)slot * LT);
  Loaded<T, G, V, LT> d;
  load_tokens<T, G, V, LT, PACKED>(p, k, ch, n, d);
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.f;
    B[v] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    float a[V], u[V];
    maps_of<FORM>(p, k, d, i, ch, n, a, u);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      B[v] = leave(a[v], u[v], B[v]);
      A[v] = drops(a[v]) ? a[v] : A[v] * a[v];
    }
  }
  sm.put(slot, c, A, B);
  __syncthreads();
  sm.compose();
  __syncthreads();
  if constexpr (PHASE == 0) {
    const int cc = threadIdx.x;
    if (cc < CB && cb * CB + cc < p.H) {
      float ta, tb;
      sm.whole(cc, ta, tb);
      p.agg_a[tile * p.H + cb * CB + cc] = ta;
      p.agg_b[tile * p.H + cb * CB + cc] = tb;
    }
  } else {
    if (n <= 0) return;
    Vec<float, V> h{};
    if (tile > 0) h = load_vec<float, V>(p.carry + tile * p.H + ch, n);
#pragma unroll
    for (int v = 0; v < V; ++v) h.v[v] = sm.enter(slot, c * V + v, h.v[v]);
    if (p.states != nullptr && k.t0 % kScanTileBwd == 0 && k.t0 < p.N)
      store_vec<float, V>(p.states + k.t0 / kScanTileBwd * p.H + ch, h, n);
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      if (k.t0 + i >= p.N) break;
      float a[V], u[V];
      maps_of<FORM>(p, k, d, i, ch, n, a, u);
      Vec<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h.v[v] = leave(a[v], u[v], h.v[v]);
        o.v[v] = (T)h.v[v];
      }
      store_vec<T, V>(static_cast<T*>(p.out) + (k.t0 + i) * p.H + ch, o, n);
      if (k.end >> i & 1) store_vec<float, V>(p.hf + (long long)k.b[i] * p.H + ch, h, n);
    }
  }
}

// What enters every tile, one thread per channel; REV for the backward's order.
template <bool REV>
__global__ __launch_bounds__(64) void scan_carry_kernel(ScanArgs p, long long ntiles) {
  const int ch = blockIdx.x * 64 + threadIdx.x;
  if (ch >= p.H) return;
  float h = 0.f;
  for (long long j = 0; j < ntiles; ++j) {
    const long long at = (REV ? ntiles - 1 - j : j) * p.H + ch;
    p.carry[at] = h;
    h = leave(p.agg_a[at], p.agg_b[at], h);
  }
}

// Backward: the carry from token t + 1 to t is a_{t+1} d_{t+1}, nothing across
// sequences.
template <class T, class G, int FORM, bool PACKED, int PHASE>
__global__ __launch_bounds__(kScanThreads) void scan_bwd_kernel(ScanArgs p, int cblocks) {
  constexpr int V = vec_of<T>(), CB = kScanLanes * V, LT = kScanTokensBwd;
  __shared__ SlotMaps<CB> sf, sr;
  const int c = threadIdx.x % kScanLanes, slot = threadIdx.x / kScanLanes;
  const long long tile = blockIdx.x / cblocks;
  const int cb = blockIdx.x % cblocks;
  const int ch = cb * CB + c * V;
  const int n = p.H - ch;
  const Tokens<LT> k = tokens_of<LT, PACKED>(p, tile * kScanTileBwd + (long long)slot * LT);
  Loaded<T, G, V, LT> d;
  load_tokens<T, G, V, LT, PACKED>(p, k, ch, n, d);
  // dL/dout, with dL/d state_final at a sequence's last token
  Vec<T, V> go[LT];
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    go[i] = Vec<T, V>{};
    if (p.go != nullptr && n > 0 && (k.valid >> i & 1))
      go[i] = load_vec<T, V>(static_cast<const T*>(p.go) + row_of<PACKED>(k, i, p.sob, p.sot) + ch, n);
  }
  auto grad_at = [&](int i, float(&o)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = (float)go[i].v[v];
    if (p.gh != nullptr && n > 0 && (k.end >> i & 1)) {
      const Vec<float, V> gh = load_vec<float, V>(p.gh + (long long)k.b[i] * p.H + ch, n);
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] += gh.v[v];
    }
  };
  float A[V], B[V], C[V], D[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = C[v] = 1.f;
    B[v] = D[v] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    float a[V], u[V];
    maps_of<FORM>(p, k, d, i, ch, n, a, u);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      B[v] = leave(a[v], u[v], B[v]);
      A[v] = drops(a[v]) ? a[v] : A[v] * a[v];
    }
  }
#pragma unroll
  for (int i = LT - 1; i >= 0; --i) {
    float a[V], u[V], o[V];
    maps_of<FORM>(p, k, d, i, ch, n, a, u);
    grad_at(i, o);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // nothing passes to the token before a sequence's first
      D[v] = drops(a[v]) ? 0.f : a[v] * (o[v] + D[v]);
      C[v] = drops(a[v]) ? a[v] : C[v] * a[v];
    }
  }
  if constexpr (PHASE == 1) sf.put(slot, c, A, B);
  sr.put(kScanSlots - 1 - slot, c, C, D);
  __syncthreads();
  if constexpr (PHASE == 1) sf.compose();
  sr.compose();
  __syncthreads();
  if constexpr (PHASE == 0) {
    const int cc = threadIdx.x;
    if (cc < CB && cb * CB + cc < p.H) {
      float ta, tb;
      sr.whole(cc, ta, tb);
      p.agg_a[tile * p.H + cb * CB + cc] = ta;
      p.agg_b[tile * p.H + cb * CB + cc] = tb;
    }
  } else {
    if (n <= 0 || k.t0 >= p.N) return;
    Vec<float, V> h = load_vec<float, V>(p.states + tile * p.H + ch, n);
    Vec<float, V> e = load_vec<float, V>(p.carry + tile * p.H + ch, n);
    float hp[LT][V];  // state before token i
#pragma unroll
    for (int v = 0; v < V; ++v) {
      hp[0][v] = sf.enter(slot, c * V + v, h.v[v]);
      e.v[v] = sr.enter(kScanSlots - 1 - slot, c * V + v, e.v[v]);
    }
#pragma unroll
    for (int i = 0; i + 1 < LT; ++i) {
      float a[V], u[V];
      maps_of<FORM>(p, k, d, i, ch, n, a, u);
#pragma unroll
      for (int v = 0; v < V; ++v) hp[i + 1][v] = leave(a[v], u[v], hp[i][v]);
    }
#pragma unroll
    for (int i = LT - 1; i >= 0; --i) {
      if (k.t0 + i >= p.N) continue;
      const bool valid = k.valid >> i & 1, start = k.start >> i & 1;
      float o[V];
      grad_at(i, o);
      Vec<float, V> h0 = start ? state_of<V>(p, k, i, ch, n) : Vec<float, V>{};
      Vec<T, V> gx;
      Vec<G, V> gg;
      Vec<float, V> gs;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, na;
        gate_of<FORM>((float)d.g[i].v[v], a, na);
        const float x = (float)d.x[i].v[v], hb = start ? h0.v[v] : hp[i][v];
        const float dt = valid ? o[v] + e.v[v] : 0.f;
        gx.v[v] = (T)(na * dt);
        if constexpr (FORM == LTC_GATE_BLEND) gg.v[v] = (G)(valid ? dt * (hb - x) * (a * na) : 0.f);
        else gg.v[v] = (G)(valid ? dt * hb * a : 0.f);
        gs.v[v] = a * dt;
        e.v[v] = start || !valid ? 0.f : gs.v[v];
      }
      const long long at = (k.t0 + i) * p.H + ch;
      if (p.gx != nullptr) store_vec<T, V>(static_cast<T*>(p.gx) + at, gx, n);
      if (p.gg != nullptr) store_vec<G, V>(static_cast<G*>(p.gg) + at, gg, n);
      if (start && p.gs != nullptr) store_vec<float, V>(p.gs + (long long)k.b[i] * p.H + ch, gs, n);
    }
  }
}

// The mark of every packed token: the last sequence that starts at or before
// it, by bisection. Any boundaries give marks in range; those of ascending
// boundaries are right.
__global__ __launch_bounds__(256) void scan_marks_kernel(const int* cu, int S, long long N, int* marks) {
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  if (t >= N) return;
  int lo = 0, hi = S + 1;  // first index whose boundary lies behind t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  const int s = lo - 1;
  int m = kMarkNone;
  if (s >= 0 && s < S)
    m = 4 * s + (cu[s] == t ? kMarkStart : 0) + (cu[s + 1] == t + 1 || t + 1 == N ? kMarkEnd : 0);
  marks[t] = m;
}

__global__ __launch_bounds__(256) void scan_empty_kernel(const int* cu, int S, int H, long long N,
                                                         const float* src, float* dst) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)S * H) return;
  const int s = (int)(i / H);
  // a sequence whose first token lies behind the tokens has none either
  const bool empty = cu == nullptr || cu[s + 1] <= cu[s] || cu[s] >= N || cu[s] < 0;
  if (empty) dst[i] = src != nullptr ? src[i] : 0.f;
}

// One token of each row, its state updated in place. A row whose slot an
// earlier row names too is left to that row, which takes the rows of its slot
// one after the other, as tokens of one stream.
template <class T, class G, int FORM>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(StepArgs p) {
  constexpr int V = vec_of<T>();
  const int row = blockIdx.y;
  const int ch = (blockIdx.x * kScanThreads + threadIdx.x) * V;
  const int n = p.H - ch;
  int slot = row;
  if (p.slots != nullptr) {
    slot = p.slots[row];
    int earlier = 0;
    for (int r = threadIdx.x; r < row; r += kScanThreads) earlier |= p.slots[r] == slot;
    const bool live = slot >= 0 && slot < p.P;
    if (!live) {
      // padding gives zeros, a slot that is not there NaN
      const float f = slot < 0 ? 0.f : __builtin_nanf("");
      Vec<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v) o.v[v] = (T)f;
      if (n > 0) store_vec<T, V>(static_cast<T*>(p.out) + (long long)row * p.H + ch, o, n);
    }
    if (__syncthreads_or(earlier) || !live) return;
  }
  if (n <= 0) return;
  float* sp = p.state + slot * p.ssp + ch;
  Vec<float, V> h = load_vec<float, V>(sp, n);
  for (int r = row; r < p.B; ++r) {
    if (r > row && (p.slots == nullptr || p.slots[r] != slot)) {
      if (p.slots == nullptr) break;
      continue;
    }
    const Vec<T, V> x = load_vec<T, V>(static_cast<const T*>(p.x) + r * p.sxb + ch, n);
    const Vec<G, V> g = load_vec<G, V>(static_cast<const G*>(p.g) + r * p.sgb + ch, n);
    Vec<T, V> o;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a, na;
      gate_of<FORM>((float)g.v[v], a, na);
      h.v[v] = fmaf(a, h.v[v], na * (float)x.v[v]);
      o.v[v] = (T)h.v[v];
    }
    store_vec<T, V>(static_cast<T*>(p.out) + (long long)r * p.H + ch, o, n);
  }
  store_vec<float, V>(sp, h, n);
}

int x_vec(int x_type) { return x_type == LTC_F32 ? 4 : 8; }

// Calls f with the element types of x and the gate.
template <class F>
hipError_t with_types(int x_type, int g_type, F&& f) {
  if (x_type == LTC_F32) return f(float{}, float{});
  if (x_type == LTC_BF16) return g_type == LTC_F32 ? f(__bf16{}, float{}) : f(__bf16{}, __bf16{});
  return g_type == LTC_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
}

template <class F>
hipError_t with_form(int form, bool packed, F&& f) {
  using std::false_type;
  using std::true_type;
  if (form == LTC_GATE_BLEND)
    return packed ? f(std::integral_constant<int, LTC_GATE_BLEND>{}, true_type{})
                  : f(std::integral_constant<int, LTC_GATE_BLEND>{}, false_type{});
  return packed ? f(std::integral_constant<int, LTC_GATE_DECAY>{}, true_type{})
                : f(std::integral_constant<int, LTC_GATE_DECAY>{}, false_type{});
}

}  // namespace

ScanPlan scan_plan(int x_type, int g_type, int form, bool packed, long long N, int H, bool bwd) {
  ScanPlan p{};
  p.x_type = x_type;
  p.g_type = g_type;
  p.form = form;
  p.packed = packed;
  p.tile = bwd ? kScanTileBwd : kScanTileFwd;
  p.ntiles = (N + p.tile - 1) / p.tile;
  const int cb = kScanLanes * x_vec(x_type);
  p.cblocks = (H + cb - 1) / cb;
  return p;
}

hipError_t launch_scan_marks(const int* cu, int S, long long N, int* marks, hipStream_t s) {
  LTC_LAUNCH(scan_marks_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s, cu, S, N, marks);
  return hipGetLastError();
}

hipError_t launch_scan_empty(const int* cu, int S, int H, long long N, const float* src, float* dst,
                             hipStream_t s) {
  const long long n = (long long)S * H;
  LTC_LAUNCH(scan_empty_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, cu, S, H, N, src,
             dst);
  return hipGetLastError();
}

hipError_t launch_scan_fwd(const ScanPlan& p, const ScanArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(p.ntiles * p.cblocks)), block(kScanThreads);
  return with_types(p.x_type, p.g_type, [&](auto t, auto g) {
    return with_form(p.form, p.packed, [&](auto form, auto packed) {
      using T = decltype(t);
      using G = decltype(g);
      constexpr int F = decltype(form)::value;
      constexpr bool P = decltype(packed)::value;
      if (p.ntiles > 1) {
        LTC_LAUNCH((scan_fwd_kernel<T, G, F, P, 0>), grid, block, 0, s, a, p.cblocks);
        LTC_LAUNCH(scan_carry_kernel<false>, dim3((a.H + 63) / 64), dim3(64), 0, s, a, p.ntiles);
      }
      LTC_LAUNCH((scan_fwd_kernel<T, G, F, P, 1>), grid, block, 0, s, a, p.cblocks);
      return hipGetLastError();
    });
  });
}

hipError_t launch_scan_bwd(const ScanPlan& p, const ScanArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(p.ntiles * p.cblocks)), block(kScanThreads);
  return with_types(p.x_type, p.g_type, [&](auto t, auto g) {
    return with_form(p.form, p.packed, [&](auto form, auto packed) {
      using T = decltype(t);
      using G = decltype(g);
      constexpr int F = decltype(form)::value;
      constexpr bool P = decltype(packed)::value;
      LTC_LAUNCH((scan_bwd_kernel<T, G, F, P, 0>), grid, block, 0, s, a, p.cblocks);
      LTC_LAUNCH(scan_carry_kernel<true>, dim3((a.H + 63) / 64), dim3(64), 0, s, a, p.ntiles);
      LTC_LAUNCH((scan_bwd_kernel<T, G, F, P, 1>), grid, block, 0, s, a, p.cblocks);
      return hipGetLastError();
    });
  });
}

hipError_t launch_scan_step(int x_type, int g_type, int form, const StepArgs& a, hipStream_t s) {
  const int per = kScanThreads * x_vec(x_type);
  const dim3 grid((unsigned)((a.H + per - 1) / per), (unsigned)a.B), block(kScanThreads);
  return with_types(x_type, g_type, [&](auto t, auto g) {
    using T = decltype(t);
    using G = decltype(g);
    if (form == LTC_GATE_BLEND)
      LTC_LAUNCH((scan_step_kernel<T, G, LTC_GATE_BLEND>), grid, block, 0, s, a);
    else
      LTC_LAUNCH((scan_step_kernel<T, G, LTC_GATE_DECAY>), grid, block, 0, s, a);
    return hipGetLastError();
  });
}

}  // namespace ltc
