// Gated linear recurrence h_t = a_t h_{t-1} + u_t per channel, for gfx950:
//   blend: a = sigmoid(g), u = (1 - a) x      decay: a = exp(g), u = x
// Its backward, with d_t = dL/dh_t + a_{t+1} d_{t+1}:
//   blend: dL/dx = (1 - a) d, dL/dg = d (h_{t-1} - x) a (1 - a)
//   decay: dL/dx = d,         dL/dg = d h_{t-1} a
//
// A run of tokens maps the state that enters it affinely, h -> A h + B, and two
// runs compose to (A2 A1, A2 B1 + B2), so time is cut into tiles: a workgroup
// reads its tile once, leaves its map for the tiles behind it, takes what enters
// it from the maps before, and runs its tokens out of its registers. The tokens of all
// sequences lie end to end; a sequence's first token gives a h0 + u whatever comes
// from before. Decays are never negative, so a map whose A has the sign bit set
// stands for one that drops what enters it, NaN and infinities too. All maps and states are fp32; out and the
// gradients are rounded to their type once, when they are stored.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/ltc_capi.h"
#include "ltc_seq_internal.h"
#include "ltc_vec.h"

namespace ltc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Marks of packed tokens: -1 behind the last sequence (and before the first),
// else 4 * sequence + 1 for its first token + 2 for its last.
constexpr int kMarkNone = -1, kMarkStart = 1, kMarkEnd = 2;

// a and 1 - a (decay: 1), each to its own relative precision: with e = exp(-g),
// a = 1 / (1 + e) and 1 - a = e a. e is kept below 2^126, where a is 2^-126 and
// 1 - a is 1; `minimum` passes a NaN on.
// exp_of is e, or in the other form a itself, from which gate_from goes on. g log2(e) is
// one rounded product, which leaves exp2 of it off by |g| 2^-24 relative. That is more
// than an ulp only where |g| is over 1: there a, or 1 - a, is small and carries the error,
// which the other side takes on times the same smallness. A product in two parts would
// cost an instruction a gate in kernels that are bound by theirs.
template <int FORM>
__device__ __forceinline__ float exp_of(float g) {
  return FORM == LTC_GATE_BLEND
             ? __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -kLog2e, 126.f))
             : __builtin_amdgcn_exp2f(g * kLog2e);
}
template <int FORM>
__device__ __forceinline__ void gate_from(float e, float& a, float& na) {
  if constexpr (FORM == LTC_GATE_BLEND) {
    a = __builtin_amdgcn_rcpf(1.f + e);
    na = e * a;
  } else {
    a = e;
    na = 1.f;
  }
}
template <int FORM>
__device__ __forceinline__ void gate_of(float g, float& a, float& na) {
  gate_from<FORM>(exp_of<FORM>(g), a, na);
}

// A thread's tokens: bit i of the masks is token i. Tokens outside all sequences
// (valid 0) drop what comes before them, as a sequence's first does.
template <int LT>
struct Tokens {
  int t0;         // first token
  unsigned valid, start, end;
  unsigned wrap;  // uniform batches: the next token is another sequence's
  int b[LT];      // sequence of token i
  long long off_b, off_t;  // uniform batches: sequence and step of the first token
};

template <int LT, bool PACKED>
__device__ __forceinline__ Tokens<LT> tokens_of(const ScanArgs& p, int t0) {
  Tokens<LT> k;
  k.t0 = t0;
  k.valid = k.start = k.end = k.wrap = 0;
  int b = 0, r = 0;
  if constexpr (!PACKED) {
    b = (int)((unsigned)t0 / (unsigned)p.T);
    r = t0 - b * p.T;
  }
  k.off_b = b;
  k.off_t = r;
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    const bool in = t0 + i < p.N;
    if constexpr (PACKED) {
      const int m = in ? p.marks[t0 + i] : kMarkNone;
      k.b[i] = m >> 2;
      if (m >= 0) {
        k.valid |= 1u << i;
        if (m & kMarkEnd) k.end |= 1u << i;
      }
      if (m < 0 || (m & kMarkStart)) k.start |= 1u << i;
    } else {
      k.b[i] = b;
      if (in) k.valid |= 1u << i;
      if (!in || r == 0) k.start |= 1u << i;
      if (++r == p.T) {
        if (in) k.end |= 1u << i;
        k.wrap |= 1u << i;
        r = 0;
        ++b;
      }
    }
  }
  return k;
}

// First and last token of packed token t's sequence s, whatever the boundaries.
__device__ __forceinline__ int begin_of(const ScanArgs& p, int s, int t) {
  const int q = p.cu[s];
  return q < 0 || q > t ? t : q;
}
__device__ __forceinline__ int end_of(const ScanArgs& p, int s, int t) {
  const long long q = (long long)p.cu[s + 1] - 1;
  return q >= p.N ? (int)p.N - 1 : q < t ? t : (int)q;
}

// n channels of the thread's tokens from a tensor of element strides sb, st; zero
// where there are none.
template <class T, int V, int LT, bool PACKED>
__device__ __forceinline__ void load_tokens(const void* base, long long sb, long long st, const ScanArgs& p,
                                            const Tokens<LT>& k, int ch, int n, Vec<T, V> (&d)[LT]) {
  const T* q = static_cast<const T*>(base) + ch;
  long long jump = 0;
  if constexpr (PACKED) {
    q += k.t0 * st;
  } else {
    q += k.off_b * sb + k.off_t * st;
    jump = sb - p.T * st;
  }
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    d[i] = Vec<T, V>{};
    if (base != nullptr && n > 0 && (k.valid >> i & 1)) d[i] = load_vec<T, V>(q, n);
    q += st;
    if (!PACKED && (k.wrap >> i & 1)) q += jump;
  }
}

// h = the state that enters token i of the thread, where it drops what comes
// before: its sequence's initial one, or 0.
template <int V, int LT>
__device__ __forceinline__ void begin_state(const ScanArgs& p, const Tokens<LT>& k, int i, int ch, int n,
                                            float (&h)[V]) {
  Vec<float, V> q{};
  if (p.h0 != nullptr && n > 0 && (k.valid >> i & 1))
    q = load_vec<float, V>(p.h0 + (long long)k.b[i] * p.H + ch, n);
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = q.get(v);
}

// Whether a map drops what enters it, and what leaves one, h having entered.
__device__ __forceinline__ bool drops(float A) { return __float_as_int(A) < 0; }
__device__ __forceinline__ float leave(float A, float B, float h) { return drops(A) ? B : fmaf(A, h, B); }

// Workgroups of the scan: kScanSlots time slots of eight lanes, which read a row's
// 128 bytes. In shared memory a lane's channels lie in places four by four, so that
// the lanes' 16-byte accesses fill the banks: side by side, eight to a lane, they
// met in the same banks for 27 of the forward's 100 us at B8 T4096 H2048.
template <class T>
struct Scan {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int kLanes = 8;
  static constexpr int kThreads = kScanSlots * kLanes;
  static constexpr int CB = kLanes * V;
  static __device__ __forceinline__ int place(int lane, int v) {
    return v / 4 * (kLanes * 4) + lane * 4 + v % 4;
  }
  static __device__ __forceinline__ int channel(int place) {
    return place % (kLanes * 4) / 4 * V + place / (kLanes * 4) * 4 + place % 4;
  }
};

// A workgroup's exchange of its slots' maps: each slot leaves the map of its
// tokens, and every slot gets the map of all slots before it.
template <class T>
struct SlotMaps {
  static constexpr int CB = Scan<T>::CB, THREADS = Scan<T>::kThreads, V = Scan<T>::V;
  static constexpr int kParts = THREADS / CB;  // threads per channel
  static constexpr int kPer = kScanSlots / kParts;  // slots per thread
  static_assert(kParts * CB == THREADS && kPer * kParts == kScanSlots, "slot split");
  float a[kScanSlots][CB], b[kScanSlots][CB];
  float pa[kParts][CB], pb[kParts][CB];

  __device__ __forceinline__ void put(int slot, int lane, const float (&A)[V], const float (&B)[V],
                                      bool dropped) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[slot][Scan<T>::place(lane, v)] = dropped ? -1.f : fabsf(A[v]);
      b[slot][Scan<T>::place(lane, v)] = B[v];
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

// ---------------------------------------------------------------------------
// What enters a tile. Workgroups take their tiles in the order in which the
// recurrence meets them (`l`: ascending forward, descending backward), by a
// counter, so that a tile's workgroup only ever waits for workgroups that have
// started before it. Each leaves its tile's map, one 64-bit word per channel that
// says by itself whether it has been written, and the last tile of every
// kScanGroup leaves the map of its group. What enters a tile then comes from the
// maps of the groups before its own and of the tiles before it in its group, from
// the tile on that holds the sequence's first token, or, up to kScanGroup tiles
// behind that, from the tiles' alone: two hops however long the sequence, and the same
// order of sums in every run. Every wait is bounded all the
// same, by the budget of the framework's other waits between workgroups: two calls
// at once on one workspace end, with NaN and the flag raised.
// ---------------------------------------------------------------------------
constexpr unsigned long long kNoWord = ~0ull;

// The device's sticky flag of waits that were given up, read and cleared by the
// host (scan_fault).
__device__ int g_scan_fault;
__device__ __forceinline__ void gave_up() {
  __hip_atomic_store(&g_scan_fault, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void put_word(unsigned long long* w, float A, float B) {
  unsigned a = __float_as_uint(A);
  if (a == 0xffffffffu) a = 0xffc00000u;  // a NaN like the empty word's
  __hip_atomic_store(w, (unsigned long long)__float_as_uint(B) << 32 | a, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

// Up to N maps' words of a channel, w[0], w[stride], ...: read at once, and again
// until each has been written.
template <int N>
struct Words {
  unsigned long long q[N];
  // w is the same for the whole workgroup, at (in words) each thread's own.
  __device__ __forceinline__ void read(const unsigned long long* w, unsigned at, unsigned stride, int n) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      q[j] = j < n ? __hip_atomic_load(w + (at + j * stride), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
  }
  __device__ __forceinline__ bool missing() const {
    bool m = false;
#pragma unroll
    for (int j = 0; j < N; ++j) m = m || q[j] == kNoWord;
    return m;
  }
  // For spin ticks of the wall clock, and kScanPolls reads (the clock goes on while a
  // process is put aside, its workgroups together). A word that does not come is itself
  // a map that gives NaN, so what hangs on it is NaN then. The wave waits as one: lane by
  // lane, the loop's own state costs the packed decays' backward two registers, which spill.
  __device__ __forceinline__ void wait(const unsigned long long* w, unsigned at, unsigned stride, int n,
                                       long long spin) {
    if (!__any(missing())) return;
    const long long t0 = wall_clock64();
    int polls = 0;
    do {
      __builtin_amdgcn_s_sleep(1);
      read(w, at, stride, n);
    } while (__any(missing()) && (++polls < kScanPolls || wall_clock64() - t0 < spin));
    if (__any(missing())) gave_up();
  }
  // (A, B) composed with the first n, in their order.
  __device__ __forceinline__ void fold(int n, float& A, float& B) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) {
        const float a = __uint_as_float((unsigned)q[j]), b = __uint_as_float((unsigned)(q[j] >> 32));
        B = leave(a, b, B);
        A = drops(a) ? a : A * a;
      }
  }
};

template <class T>
struct LookBack {
  static constexpr int CB = Scan<T>::CB, THREADS = Scan<T>::kThreads;
  static constexpr int kParts = THREADS / CB;
  static constexpr int kTiles = kScanGroup / kParts;  // a part's share of a group
  static constexpr int kGroups = 4;  // words of a batch: more cost registers, and those spill
  float ta[kParts][CB], tb[kParts][CB], ga[kParts][CB], gb[kParts][CB];
  // The workgroup's number in order, before run(); what enters the tile, after it. No
  // places of their own: so four workgroups of the 16-bit backward fill a CU's 160 KiB.
  __device__ __forceinline__ unsigned& ticket() { return *reinterpret_cast<unsigned*>(&ta[0][0]); }
  __device__ __forceinline__ float& enter(int c) { return ga[0][c]; }

  // Leaves the tile's map (A, B: valid in threads below CB) and what enters the
  // tile, in enter(). `first`: the tile from which on maps count, l for none.
  __device__ __forceinline__ void run(const ScanArgs& p, int l, int first, int c0, float A, float B) {
    const int c = threadIdx.x % CB, part = threadIdx.x / CB;
    const int ch = Scan<T>::channel(c);
    const bool in = c0 + ch < p.H;
    const long long H = p.H;
    unsigned long long* w = p.words + c0;
    if (part == 0 && in) put_word(w + l * H + ch, A, B);
    const int g = l / kScanGroup, g0 = g * kScanGroup;
    unsigned long long* gw = p.words + p.ntiles * H + c0;
    const bool last = l == g0 + kScanGroup - 1;
    // the tiles before this one from `first` on, where they are few, or those in its
    // group, which the group's map takes all of
    const bool near = !last && l - first <= kScanGroup;
    const int from = near ? first : g0;
    const int nt = in ? l - from : 0, t0 = part * kTiles, tn = nt - t0 < kTiles ? nt - t0 : kTiles;
    // the groups before it, each part an equal share, in batches
    const int gf = first / kScanGroup;
    const int ng = in && !near && first < g0 ? g - gf : 0, per = (ng + kParts - 1) / kParts, i0 = part * per;
    const int gn = ng - i0 < per ? ng - i0 : per;
    const unsigned long long* wt = w + from * H;
    const unsigned long long* wg = gw + gf * H;
    const unsigned at = (unsigned)t0 * p.H + ch, ag = (unsigned)i0 * p.H + ch;
    Words<kTiles> qt;
    Words<kGroups> qg;
    qt.read(wt, at, p.H, tn);
    qg.read(wg, ag, p.H, gn);
    float a = 1.f, b = 0.f;
    qt.wait(wt, at, p.H, tn, p.spin);
    qt.fold(tn, a, b);
    ta[part][c] = a;
    tb[part][c] = b;
    // The group's map goes out before this tile waits for other groups': groups
    // never wait for one another in a row.
    if (last) {
      __syncthreads();
      if (part == 0 && in) {
        a = 1.f;
        b = 0.f;
        join(ta, tb, c, a, b);
        put_word(gw + g * H + ch, drops(A) ? A : a * A, leave(A, B, b));
      }
    }
    a = 1.f;
    b = 0.f;
    qg.wait(wg, ag, p.H, gn, p.spin);
    qg.fold(gn, a, b);
    for (int i = kGroups; i < gn; i += kGroups) {
      const unsigned ai = ag + (unsigned)i * p.H;
      qg.read(wg, ai, p.H, gn - i);
      qg.wait(wg, ai, p.H, gn - i, p.spin);
      qg.fold(gn - i, a, b);
    }
    ga[part][c] = a;
    gb[part][c] = b;
    __syncthreads();
    if (part == 0) {
      a = 1.f;
      b = 0.f;
      join(ga, gb, c, a, b);
      join(ta, tb, c, a, b);
      // without a budget every wait counts as given up
      if (first != l && p.spin <= 0) gave_up();
      enter(c) = first == l ? 0.f : p.spin > 0 ? b : __builtin_nanf("");
    }
    __syncthreads();
  }

  static __device__ __forceinline__ void join(const float (&pa)[kParts][CB], const float (&pb)[kParts][CB],
                                              int c, float& A, float& B) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      B = leave(pa[q][c], pb[q][c], B);
      A = drops(pa[q][c]) ? pa[q][c] : A * pa[q][c];
    }
  }
};

struct NoLookBack {};

// A workgroup's tile, in order, and its block of channels. Blocks of channels are
// dealt out in up to kScanRanges ranges of p.per side by side, one range to a
// workgroup number modulo their count, so that neighbours on a row, which may share
// lines of it, are worked on at about the same time. A counter takes one addition in
// about 15 ns, so each range has its own: one for all held B8 T4096 H2048 (8192 tiles)
// to 128 us, and one for each block let neighbours drift apart (H2047 181 us). Seven
// ranges, not eight: with one to an XCD each XCD keeps to the same few memory channels
// where rows are powers of two (H2048 forward 95 us and 103, one tile a sequence 76
// and 83).
template <bool LOOK, class LB>
__device__ __forceinline__ void take_tile(const ScanArgs& p, LB& lb, int& tile, int& cblock) {
  const unsigned range = blockIdx.x % p.ranges;
  unsigned t = blockIdx.x / p.ranges;
  if constexpr (LOOK) {
    if (threadIdx.x == 0)
      lb.ticket() = __hip_atomic_fetch_add(p.tickets + range * kTicketStride, 1u, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    t = lb.ticket();
  }
  tile = t / p.per;
  cblock = range * p.per + t % p.per;
}

// The compiler forgets what it has computed from r: it computes that again later,
// and keeps only r in registers meanwhile.
template <class T, int V, int LT>
__device__ __forceinline__ void forget(Vec<T, V> (&r)[LT]) {
#pragma unroll
  for (int i = 0; i < LT; ++i)
#pragma unroll
    for (int j = 0; j < Vec<T, V>::kWords; ++j) asm volatile("" : "+v"(r[i].w[j]));
}
template <int V, int LT>
__device__ __forceinline__ void forget(float (&r)[LT][V]) {
#pragma unroll
  for (int i = 0; i < LT; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) asm volatile("" : "+v"(r[i][v]));
}

// LOOK: tiles hand states on; else every tile begins with a sequence, or is the
// only one. B8 T4096 H2048 bf16 takes 96 us, 4.2 TB/s, and without handing on (T128) 77,
// 5.2: bound by bytes, arithmetic (formed twice, the gates cost bf16 9 us more) and the
// wait. The four workgroups that a CU holds cover one another's waits.
template <class T, class G, int FORM, bool PACKED, bool LOOK>
__global__ __launch_bounds__(Scan<T>::kThreads, 4) void scan_fwd_kernel(ScanArgs p) {
  constexpr int V = Scan<T>::V, CB = Scan<T>::CB, LT = kScanTokens;
  __shared__ SlotMaps<T> sm;
  __shared__ typename std::conditional<LOOK, LookBack<T>, NoLookBack>::type lb;
  const int c = threadIdx.x % Scan<T>::kLanes, slot = threadIdx.x / Scan<T>::kLanes;
  int tile, cblock;
  take_tile<LOOK>(p, lb, tile, cblock);
  if (cblock >= p.cblocks) return;  // the last range may be short
  const int c0 = cblock * CB, ch = c0 + c * V, n = p.H - ch;
  const Tokens<LT> k = tokens_of<LT, PACKED>(p, tile * kScanTile + slot * LT);
  // after token i, h = A[i] h_in + B[i], of the state that enters the slot
  float A[LT][V], B[LT][V];
  {
    Vec<T, V> x[LT];
    Vec<G, V> g[LT];
    load_tokens<T, V, LT, PACKED>(p.x, p.sxb, p.sxt, p, k, ch, n, x);
    load_tokens<G, V, LT, PACKED>(p.g, p.sgb, p.sgt, p, k, ch, n, g);
    float pa[V], pb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      pa[v] = 1.f;
      pb[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      if (k.start >> i & 1) {
        begin_state<V>(p, k, i, ch, n, pb);
#pragma unroll
        for (int v = 0; v < V; ++v) pa[v] = 0.f;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, na;
        gate_of<FORM>(g[i].get(v), a, na);
        const float xv = x[i].get(v);
        pa[v] *= a;
        pb[v] = fmaf(a, pb[v], FORM == LTC_GATE_BLEND ? na * xv : xv);
        A[i][v] = pa[v];
        B[i][v] = pb[v];
      }
    }
  }
  sm.put(slot, c, A[LT - 1], B[LT - 1], k.start != 0);
  __syncthreads();
  sm.compose();
  __syncthreads();
  if constexpr (LOOK) {
    // the tile of the first token's sequence's beginning
    const int t0 = tile * kScanTile;
    int first = tile;
    if constexpr (PACKED) {
      const int m = p.marks[t0];
      if (m >= 0 && !(m & kMarkStart)) first = begin_of(p, m >> 2, t0) / kScanTile;
    } else {
      const int q = t0 - (int)((unsigned)t0 % (unsigned)p.T);
      if (q < t0) first = q / kScanTile;
    }
    float ta = 1.f, tb = 0.f;
    if (threadIdx.x < CB) sm.whole(threadIdx.x, ta, tb);
    lb.run(p, tile, first, c0, ta, tb);
  }
  if (n <= 0) return;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = Scan<T>::place(c, v);
    float enter = 0.f;
    if constexpr (LOOK) enter = lb.enter(at);
    h[v] = sm.enter(slot, at, enter);
  }
  // the backward starts its tiles from these
  if (p.states != nullptr && slot == 0) {
    Vec<float, V> q;
    q.put(h);
    store_vec<float, V>(p.states + (long long)tile * p.H + ch, q, n);
  }
  T* out = static_cast<T*>(p.out) + (long long)k.t0 * p.H + ch;
#pragma unroll
  for (int i = 0; i < LT; ++i) {
    if (k.t0 + i >= p.N) break;
    if (k.start >> i & 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = 0.f;  // A[i] is 0 from here on
    }
    float o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = fmaf(A[i][v], h[v], B[i][v]);
    Vec<T, V> q;
    q.put(o);
    store_vec<T, V>(out, q, n);
    out += p.H;
    if (k.end >> i & 1) {
      Vec<float, V> f;
      f.put(o);
      store_vec<float, V>(p.hf + (long long)k.b[i] * p.H + ch, f, n);
    }
  }
}

// Backward: the carry from token t + 1 to t is a_{t+1} d_{t+1}, nothing across
// sequences. The states are run again from what entered the tile. Gates are formed
// three times (for the maps, the states, the gradients): kept, they take 64
// registers more, which spill. Of 16-bit inputs their exponentials are kept, in 16
// registers more: the kernel is bound by its arithmetic there as much as by its bytes
// (B8 T4096 H2048 bf16 175 us and 185, 3.8 TB/s). In fp32, with half the arithmetic to
// a byte, it runs faster without (H1024 159 us and 173, 4.2 TB/s).
// Decays need fewer registers, 128 of them: four workgroups to a CU for three (with the
// preparation, B8 T4096 H2048 bf16 140 us and 152; 30011 tokens in 37 sequences, H1000
// bf16, fp32 gates 137 and 141).
template <class T, class G, int FORM, bool PACKED, bool LOOK>
__global__ __launch_bounds__(Scan<T>::kThreads, sizeof(T) == 2 && FORM == LTC_GATE_DECAY ? 4 : 3)
    void scan_bwd_kernel(ScanArgs p) {
  constexpr int V = Scan<T>::V, CB = Scan<T>::CB, LT = kScanTokens;
  __shared__ SlotMaps<T> sf, sr;
  __shared__ typename std::conditional<LOOK, LookBack<T>, NoLookBack>::type lb;
  const int c = threadIdx.x % Scan<T>::kLanes, slot = threadIdx.x / Scan<T>::kLanes;
  int l, cblock;
  take_tile<LOOK>(p, lb, l, cblock);
  if (cblock >= p.cblocks) return;  // the last range may be short
  const int tile = (int)p.ntiles - 1 - l;
  const int c0 = cblock * CB, ch = c0 + c * V, n = p.H - ch;
  const Tokens<LT> k = tokens_of<LT, PACKED>(p, tile * kScanTile + slot * LT);
  Vec<T, V> x[LT], go[LT];
  Vec<G, V> g[LT];
  constexpr bool KEEP = sizeof(T) == 2;
  float ex[LT][V];  // KEEP: exp_of the gates, else the gates
  auto gate = [&](int i, int v, float& a, float& na) {
    if constexpr (KEEP) gate_from<FORM>(ex[i][v], a, na);
    else gate_of<FORM>(ex[i][v], a, na);
  };
  load_tokens<T, V, LT, PACKED>(p.x, p.sxb, p.sxt, p, k, ch, n, x);
  load_tokens<G, V, LT, PACKED>(p.g, p.sgb, p.sgt, p, k, ch, n, g);
  load_tokens<T, V, LT, PACKED>(p.go, p.sob, p.sot, p, k, ch, n, go);
  // o += dL/d state_final, at a sequence's last token
  auto add_end = [&](int i, float(&o)[V]) {
    if (p.gh == nullptr || n <= 0 || !(k.end >> i & 1)) return;
    const Vec<float, V> gh = load_vec<float, V>(p.gh + (long long)k.b[i] * p.H + ch, n);
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] += gh.get(v);
  };
  {
    // the map of the slot's tokens, and of the carries through them
    float a[LT][V], A[V], B[V], D[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] = 1.f;
      B[v] = D[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      if (k.start >> i & 1) begin_state<V>(p, k, i, ch, n, B);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float na;
        ex[i][v] = KEEP ? exp_of<FORM>(g[i].get(v)) : g[i].get(v);
        gate(i, v, a[i][v], na);
        const float xv = x[i].get(v);
        A[v] *= a[i][v];
        B[v] = fmaf(a[i][v], B[v], FORM == LTC_GATE_BLEND ? na * xv : xv);
      }
    }
#pragma unroll
    for (int i = LT - 1; i >= 0; --i) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = go[i].get(v);
      add_end(i, o);
#pragma unroll
      for (int v = 0; v < V; ++v) D[v] = a[i][v] * (o[v] + D[v]);
      if (k.start >> i & 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) D[v] = 0.f;
      }
    }
    sf.put(slot, c, A, B, k.start != 0);
    sr.put(kScanSlots - 1 - slot, c, A, D, k.start != 0);
  }
  __syncthreads();
  sf.compose();
  sr.compose();
  __syncthreads();
  if constexpr (LOOK) {
    // the tile of the end of the last token's sequence
    const int t1 = tile * kScanTile + kScanTile - 1 < p.N ? tile * kScanTile + kScanTile - 1 : (int)p.N - 1;
    int first = l;
    if constexpr (PACKED) {
      const int m = p.marks[t1];
      if (m >= 0 && !(m & kMarkEnd)) first = (int)p.ntiles - 1 - end_of(p, m >> 2, t1) / kScanTile;
    } else {
      const int q = t1 - (int)((unsigned)t1 % (unsigned)p.T) + p.T - 1;
      if (q > t1) first = (int)p.ntiles - 1 - q / kScanTile;
    }
    float ta = 1.f, tb = 0.f;
    if (threadIdx.x < CB) sr.whole(threadIdx.x, ta, tb);
    lb.run(p, l, first, c0, ta, tb);
  }
  forget(x);
  forget(ex);
  forget(go);
  if (n <= 0 || k.t0 >= p.N) return;
  float hp[LT][V], e[V];  // state before token i, carry into it
  {
    const Vec<float, V> q = load_vec<float, V>(p.states + (long long)tile * p.H + ch, n);
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = Scan<T>::place(c, v);
      h[v] = sf.enter(slot, at, q.get(v));
      float enter = 0.f;
      if constexpr (LOOK) enter = lb.enter(at);
      e[v] = sr.enter(kScanSlots - 1 - slot, at, enter);
    }
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      if (k.start >> i & 1) begin_state<V>(p, k, i, ch, n, h);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, na;
        gate(i, v, a, na);
        const float xv = x[i].get(v);
        hp[i][v] = h[v];
        h[v] = fmaf(a, h[v], FORM == LTC_GATE_BLEND ? na * xv : xv);
      }
    }
  }
  forget(ex);
  long long at = (long long)k.t0 * p.H + ch + (LT - 1) * (long long)p.H;
#pragma unroll
  for (int i = LT - 1; i >= 0; --i, at -= p.H) {
    if (k.t0 + i >= p.N) continue;
    float o[V], dx[V], dg[V], ds[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = go[i].get(v);
    add_end(i, o);
    if (!(k.valid >> i & 1)) {
#pragma unroll
      for (int v = 0; v < V; ++v) e[v] = hp[i][v] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a, na;
      gate(i, v, a, na);
      const float d = o[v] + e[v];
      e[v] = ds[v] = a * d;
      if constexpr (FORM == LTC_GATE_BLEND) {
        dx[v] = na * d;
        dg[v] = ds[v] * (na * (hp[i][v] - x[i].get(v)));
      } else {
        dx[v] = d;
        dg[v] = ds[v] * hp[i][v];
      }
    }
    if (p.gx != nullptr) {
      Vec<T, V> q;
      q.put(dx);
      store_vec<T, V>(static_cast<T*>(p.gx) + at, q, n);
    }
    if (p.gg != nullptr) {
      Vec<G, V> q;
      q.put(dg);
      store_vec<G, V>(static_cast<G*>(p.gg) + at, q, n);
    }
    if (k.start >> i & 1) {
      if (p.gs != nullptr && (k.valid >> i & 1)) {
        Vec<float, V> q;
        q.put(ds);
        store_vec<float, V>(p.gs + (long long)k.b[i] * p.H + ch, q, n);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) e[v] = 0.f;
    }
  }
}

// Before the scan: no words, the first tiles' tickets; for packed tokens their marks (the
// last sequence that starts at or before a token, by bisection: any boundaries
// give marks in range, ascending ones the right ones), and dst = src for the
// empty sequences, which no token writes (all of them without tokens).
__global__ __launch_bounds__(256) void scan_prep_kernel(ScanPrep p) {
  const long long i0 = (long long)blockIdx.x * 256 + threadIdx.x, step = (long long)gridDim.x * 256;
  for (long long i = i0; i < p.nwords; i += step) p.words[i] = kNoWord;
  if (p.tickets != nullptr && i0 < kScanRanges) p.tickets[i0 * kTicketStride] = 0;
  if (p.marks != nullptr)
    for (long long t = i0; t < p.N; t += step) {
      int lo = 0, hi = p.S + 1;  // first index whose boundary lies behind t
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.cu[mid] <= t) lo = mid + 1;
        else hi = mid;
      }
      const int s = lo - 1;
      int m = kMarkNone;
      if (s >= 0 && s < p.S)
        m = 4 * s + (p.cu[s] == t ? kMarkStart : 0) + (p.cu[s + 1] == t + 1 || t + 1 == p.N ? kMarkEnd : 0);
      p.marks[t] = m;
    }
  if (p.dst != nullptr)
    for (long long i = i0; i < (long long)p.S * p.H; i += step) {
      const int s = (int)(i / p.H);
      // a sequence that begins outside the tokens has none either
      const bool empty = p.N == 0 || p.cu[s + 1] <= p.cu[s] || p.cu[s] >= p.N || p.cu[s] < 0;
      if (empty) p.dst[i] = p.src != nullptr ? p.src[i] : 0.f;
    }
}

constexpr int kStepThreads = 256, kStepChannels = 4;

// One token of each row, its state updated in place. A row whose slot an
// earlier row names too is left to that row, which takes the rows of its slot
// one after the other, as tokens of one stream. Bound by latency: the loads are
// under way before the workgroup has looked through the slots for its own (one row of
// 64 1.5 us, 256 rows of 2048 in a pool 4.0).
template <class T, class G, int FORM>
__global__ __launch_bounds__(kStepThreads) void scan_step_kernel(StepArgs p) {
  constexpr int V = kStepChannels;
  const int row = blockIdx.y;
  const int ch = (blockIdx.x * kStepThreads + threadIdx.x) * V;
  const int n = p.H - ch;
  const int slot = p.slots != nullptr ? p.slots[row] : row;
  const bool live = slot >= 0 && slot < p.P;
  Vec<T, V> x{};
  Vec<G, V> g{};
  Vec<float, V> s{};
  if (n > 0 && live) {
    x = load_vec<T, V>(static_cast<const T*>(p.x) + row * p.sxb + ch, n);
    g = load_vec<G, V>(static_cast<const G*>(p.g) + row * p.sgb + ch, n);
    s = load_vec<float, V>(p.state + slot * p.ssp + ch, n);
  }
  T* out = static_cast<T*>(p.out) + ch;
  int more = 0;  // whether later rows name the slot
  if (p.slots != nullptr) {
    int earlier = 0;
    for (int r = threadIdx.x; r < p.B; r += kStepThreads) {
      const bool same = p.slots[r] == slot;
      earlier |= same && r < row;
      more |= same && r > row;
    }
    earlier = __syncthreads_or(earlier);
    more = __syncthreads_or(more);
    if (!live) {
      // padding gives zeros, a slot that is not there NaN
      float f[V];
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = slot < 0 ? 0.f : __builtin_nanf("");
      Vec<T, V> o;
      o.put(f);
      if (n > 0) store_vec<T, V>(out + (long long)row * p.H, o, n);
      return;
    }
    if (earlier) return;
  }
  if (n <= 0) return;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = s.get(v);
  auto step = [&](int r) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a, na;
      gate_of<FORM>(g.get(v), a, na);
      h[v] = fmaf(a, h[v], na * x.get(v));
    }
    Vec<T, V> o;
    o.put(h);
    store_vec<T, V>(out + (long long)r * p.H, o, n);
  };
  step(row);
  if (more)
    for (int r = row + 1; r < p.B; ++r) {
      if (p.slots[r] != slot) continue;
      x = load_vec<T, V>(static_cast<const T*>(p.x) + r * p.sxb + ch, n);
      g = load_vec<G, V>(static_cast<const G*>(p.g) + r * p.sgb + ch, n);
      step(r);
    }
  s.put(h);
  store_vec<float, V>(p.state + slot * p.ssp + ch, s, n);
}

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

void scan_tiles(int x_type, long long N, int H, ScanArgs* a) {
  const int cb = x_type == LTC_F32 ? Scan<float>::CB : Scan<__bf16>::CB;
  a->ntiles = (N + kScanTile - 1) / kScanTile;
  a->cblocks = (H + cb - 1) / cb;
  // At least 512 bytes of a row side by side where there are as many: H512 T131072
  // forward 112 us, with blocks dealt out singly 125. Where all workgroups run at once
  // (the backward's: nearly) they cannot drift far apart, and a counter for every block gets them started sooner:
  // B4 T1999 H320 fp16 12.6 us and 14.3.
  a->per = (a->cblocks + kScanRanges - 1) / kScanRanges;
  const bool at_once = a->cblocks <= kScanRanges && a->ntiles * a->cblocks <= 1024;
  if (a->per < 4 && !at_once) a->per = a->cblocks < 4 ? a->cblocks : 4;
  a->ranges = (a->cblocks + a->per - 1) / a->per;
}

// Whether states pass from tile to tile.
bool scan_looks(long long N, int T, bool packed) {
  return N > kScanTile && (packed || kScanTile % T != 0);
}

hipError_t launch_scan_prep(const ScanPrep& p, hipStream_t s) {
  long long n = p.nwords;
  if (p.marks != nullptr && p.N > n) n = p.N;
  if (p.dst != nullptr && (long long)p.S * p.H > n) n = (long long)p.S * p.H;
  const long long blocks = (n + 255) / 256;
  LTC_LAUNCH(scan_prep_kernel, dim3((unsigned)(blocks < 1 ? 1 : blocks > 2048 ? 2048 : blocks)), dim3(256),
             0, s, p);
  return hipGetLastError();
}

hipError_t launch_scan(const ScanTypes& ty, const ScanArgs& a, bool bwd, hipStream_t s) {
  const dim3 grid((unsigned)(a.ntiles * a.per * a.ranges));
  const bool look = scan_looks(a.N, a.T, a.marks != nullptr);
  return with_types(ty.x, ty.g, [&](auto t, auto g) {
    return with_form(ty.form, a.marks != nullptr, [&](auto form, auto packed) {
      using T = decltype(t);
      using G = decltype(g);
      const dim3 block(Scan<T>::kThreads);
      constexpr int F = decltype(form)::value;
      constexpr bool P = decltype(packed)::value;
      if (bwd) {
        if (look) LTC_LAUNCH((scan_bwd_kernel<T, G, F, P, true>), grid, block, 0, s, a);
        else LTC_LAUNCH((scan_bwd_kernel<T, G, F, P, false>), grid, block, 0, s, a);
      } else {
        if (look) LTC_LAUNCH((scan_fwd_kernel<T, G, F, P, true>), grid, block, 0, s, a);
        else LTC_LAUNCH((scan_fwd_kernel<T, G, F, P, false>), grid, block, 0, s, a);
      }
      return hipGetLastError();
    });
  });
}

hipError_t scan_fault(int* value, bool clear) {
  return read_flag(&g_scan_fault, value, clear);
}

hipError_t launch_scan_step(int x_type, int g_type, int form, const StepArgs& a, hipStream_t s) {
  const int per = kStepThreads * kStepChannels;
  const dim3 grid((unsigned)((a.H + per - 1) / per), (unsigned)a.B), block(kStepThreads);
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
