// Selective state space scan, for gfx950. Of every channel c and state n:
//   D_t = delta_t (+ bias), or softplus of it      a = exp(D_t A[c,n])
//   h_t = a h_{t-1} + D_t B_t[n] x_t               y_t = sum_n C_t[n] h_t + skip x_t
//   out_t = y_t, or y_t silu(z_t)
// Backward, with dy = dout or dout silu(z) and d_t = C_t dy_t + a_{t+1} d_{t+1}:
//   dL/dB_t[n] = sum_c d D x      dL/dC_t[n] = sum_c dy h      s1 = sum_n d B
//   dL/dx = D s1 + skip dy        dL/dD = x s1 + sum_n A a h_{t-1} d
//   dL/dA = sum_t D a h_{t-1} d
//
// Arithmetic bounds it: forward a product, an exponential (twice a product's time), a
// product and two multiply-adds a state; backward these once more and about twelve, and what
// it takes to sum over channels. A product with a scalar or a lane-crossing operand takes
// 4.4 cycles, one of a lane's own registers 2.4 if another wave shares the SIMD, and one
// wave alone issues one in 4.4: measured.
//
// The forward gives a channel four lanes, each with four states, so waves need nothing of
// one another. The backward gives it one lane of each of eight waves, each with two states;
// step sizes are formed once and handed round in shared memory, the waves' sums over states
// go the same way, and the sums over channels, for dB and dC, are formed by halving: 64
// sums over 64 lanes take 63 exchanges instead of 384. (The backward with four lanes a
// channel was built too: 837 us for 787 at B8 T2048 H2048 N16, since its decays, states and
// sums need 370 registers.) Both walk a chunk of the time axis in batches of 16 tokens, the
// next batch's inputs under way.
//
// The forward leaves the states before every batch for the backward. Sequences that are
// too few to fill the chip are cut into chunks: a first launch runs each chunk from
// nothing, a second one puts what leaves them together, since the decays of a chunk have
// the product exp(A sum D), and the walk itself then starts from what enters. All states
// and sums are fp32, in an order that the sizes alone decide.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/ltc_capi.h"
#include "ltc_model_internal.h"
#include "ltc_tokens.h"
#include "ltc_vec.h"

namespace ltc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kL = kSsmTokens;
constexpr unsigned kAll = (1u << kL) - 1;

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + exp2_of(v * -kLog2e));
}

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|). With w = 1 + e rounded, the
// logarithm is log(w) e / (w - 1): the rounding of w cancels, so small e keep their
// precision (Higham, Accuracy and Stability of Numerical Algorithms, 1.14.1).
__device__ __forceinline__ float softplus(float v) {
  const float e = exp2_of(fabsf(v) * -kLog2e);
  const float w = 1.f + e, f = w - 1.f;
  constexpr float kLn2 = 0.6931471805599453f;
  const float l = f == 0.f ? e : __builtin_amdgcn_logf(w) * (kLn2 * e * __builtin_amdgcn_rcpf(f));
  return fmaxf(v, 0.f) + l;
}

// Element `i` of a row that is the same for the wave: a 32-bit offset of the lane's own
// leaves the row's address to the scalar unit.
template <class T>
__device__ __forceinline__ T& lane_of(T* row, int i) {
  return *reinterpret_cast<T*>(const_cast<char*>(reinterpret_cast<const char*>(row)) + (unsigned)i * (unsigned)sizeof(T));
}

// A value that has arrived. A load that is still under way where branches or a loop's
// rounds join would be waited for at its use in every round, and with it all later ones.
__device__ __forceinline__ void settle(float& v) { asm volatile("" : "+v"(v)); }

// The initial states of sequences without tokens are their final ones.
__global__ __launch_bounds__(256) void ssm_empty_kernel(SsmArgs p, const float* src, float* dst) {
  const long long hn = (long long)p.H * p.N;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.B * hn; i += (long long)gridDim.x * 256) {
    int lo = 0, hi = 0;
    if (p.ntok > 0) span_of(p.cu, p.T, (int)p.ntok, (int)(i / hn), lo, hi);
    if (lo == hi) dst[i] = src != nullptr ? src[i] : 0.f;
  }
}

// ---------------------------------------------------------------------------
// What the walks share
// ---------------------------------------------------------------------------
// A workgroup's chunk and channels.
struct Work {
  long long chunk;
  int g, hb, wave, lane;
  int c0, c1;    // tokens
  int first;     // the line's first
  int ch;        // channel of the lane
  bool in;       // whether there is one
  long long b;   // batches: the sequence
  __device__ __forceinline__ Work(const SsmArgs& p) {
    const unsigned per = (unsigned)(p.G * p.hblocks);
    chunk = blockIdx.x / per;
    const int r = (int)(blockIdx.x - chunk * per);
    g = r / p.hblocks;
    hb = r - g * p.hblocks;
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    lane = threadIdx.x % 64;
    b = chunk / p.chunks;
    first = (int)(b * p.T);
    const long long from = first + (chunk - b * p.chunks) * (long long)p.len, last = (long long)first + p.T;
    c0 = (int)from;
    c1 = (int)(from + p.len < last ? from + p.len : last);
    const int hpg = p.H / p.G;
    in = hb * 64 + lane < hpg;
    ch = g * hpg + hb * 64 + lane;
  }
  // Element of token 0 of a tensor of strides sb, st, from which the chunk's tokens count.
  __device__ __forceinline__ long long off(const SsmArgs& p, long long sb, long long st) const {
    return p.cu == nullptr ? b * (sb - p.T * st) : 0;
  }
};

using Edges = EdgesOf<kL>;
__device__ __forceinline__ int lowest(unsigned m) { return __ffs((int)m) - 1; }
__device__ __forceinline__ int highest(unsigned m) { return 31 - __clz((int)m); }
// Calls f with the offset of the states of the sequence that token t begins or ends.
template <class F>
__device__ __forceinline__ void at_state(const SsmArgs& p, int t, F&& f) {
  at_edge(p.cu, p.B, p.T, (int)p.ntok, t, [&](int s) { f((long long)s * p.H * p.N); });
}

// The E states from the q-th E of a lane's channel in (rows,H,N), n of them there.
template <int E, class F>
__device__ __forceinline__ void states(const SsmArgs& p, const Work& w, int q, F&& f) {
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (w.in && q * E + e < p.N) f(e, (long long)w.ch * p.N + q * E + e);
}
template <int E>
__device__ __forceinline__ void read_states(const SsmArgs& p, const Work& w, int q, const float* from, int t,
                                            float (&h)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) h[e] = 0.f;
  if (from == nullptr) return;
  at_state(p, t, [&](long long s) { states<E>(p, w, q, [&](int e, long long at) { h[e] = from[s + at]; }); });
#pragma unroll
  for (int e = 0; e < E; ++e) settle(h[e]);
}
// log2(e) A of E states, of the last one for those behind it.
template <int E>
__device__ __forceinline__ void read_rates(const SsmArgs& p, const Work& w, int q, float (&A2)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    A2[e] = w.in ? p.A[(long long)w.ch * p.N + min(q * E + e, p.N - 1)] * kLog2e : 0.f;
    settle(A2[e]);
  }
}

// A wave's tokens of a batch, wave, wave + waves, ..., at most M of them: their inputs,
// which wait in registers, as they were read, until the batch is at hand. Where there is
// no token or channel another one's are read: a branch would wait for each by itself.
template <class T, int M>
struct Inputs {
  T x[M], d[M], z[M], go[M];
  template <bool BWD>
  __device__ __forceinline__ void load(const SsmArgs& p, const Work& w, int waves, int t) {
    const int ch = w.in ? w.ch : w.g * (p.H / p.G);
    const T* px = static_cast<const T*>(p.x) + w.off(p, p.sxb, p.sxt);
    const T* pd = static_cast<const T*>(p.d) + w.off(p, p.sdb, p.sdt);
    const T* pz = static_cast<const T*>(p.z) + w.off(p, p.szb, p.szt);
    const T* pg = static_cast<const T*>(p.go) + (BWD ? w.off(p, p.sob, p.sot) : 0);
    long long u[M];
#pragma unroll
    for (int j = 0; j < M; ++j) {
      u[j] = min(t + w.wave + j * waves, w.c1 - 1);
      x[j] = lane_of(px + u[j] * p.sxt, ch);
      d[j] = lane_of(pd + u[j] * p.sdt, ch);
      z[j] = go[j] = T{};
    }
    if (p.z != nullptr) {
#pragma unroll
      for (int j = 0; j < M; ++j) z[j] = lane_of(pz + u[j] * p.szt, ch);
    }
    if (BWD && p.go != nullptr) {
#pragma unroll
      for (int j = 0; j < M; ++j) go[j] = lane_of(pg + u[j] * p.sot, ch);
    }
  }
};

// Calls f with 0 ... N-1 as constants.
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (N > 1) each<N - 1>(f);
  f(std::integral_constant<int, N - 1>{});
}
// A batch's tokens, as constants, in reverse.
template <class F>
__device__ __forceinline__ void back(F&& f) {
  each<kL>([&](auto i) { f(std::integral_constant<int, kL - 1 - decltype(i)::value>{}); });
}

// B and C of a batch and a wave's E states. They are the same for all lanes, so each row of
// 16 lanes holds all of them in kL * 2 E / 16 registers, and instructions take them from a
// lane of the row: as fast as a scalar operand, with no scalar loads to wait for. A token's
// 2 E values lie side by side.
template <class T, int E>
struct Coeffs {
  static constexpr int kToken = 2 * E, kTokens = 16 / kToken, kRegs = kL / kTokens;
  T raw[kRegs];
  float v[kRegs];
  // Of the batch at t, which wait as they were read until it is at hand (arrive).
  __device__ __forceinline__ void load(const SsmArgs& p, const Work& w, int q, int t) {
    const int k = w.lane % 16, c = k % kToken, n = min(q * E + c % E, p.N - 1);
    const bool isC = c >= E;
    const long long st = isC ? p.sct : p.sbt;
    const T* from = static_cast<const T*>(isC ? p.Cm : p.Bm) + (isC ? w.off(p, p.scb, p.sct) : w.off(p, p.sbb, p.sbt)) +
                    w.g * (isC ? p.scg : p.sbg) + n;
    if (t + kL <= w.c1) {
      from += (t + k / kToken) * st;
      const long long step = kTokens * st;
#pragma unroll
      for (int j = 0; j < kRegs; ++j, from += step) raw[j] = *from;
    } else {
#pragma unroll
      for (int j = 0; j < kRegs; ++j) raw[j] = from[min(t + j * kTokens + k / kToken, w.c1 - 1) * st];
    }
  }
  // Zero for tokens that are not in seg. States behind the last are it once more, with a C
  // of zero: they stay finite where it does, and nothing comes of them.
  __device__ __forceinline__ void arrive(const SsmArgs& p, const Work& w, int q, unsigned seg) {
    const int k = w.lane % 16, c = k % kToken;
    const bool no = c >= E && q * E + c - E >= p.N;
    const unsigned mine = no ? 0u : seg >> (k / kToken);
#pragma unroll
    for (int j = 0; j < kRegs; ++j) v[j] = mine >> (j * kTokens) & 1 ? (float)raw[j] : 0.f;
  }
  template <int I, int C>
  __device__ __forceinline__ float at() const {
    constexpr int kRowBroadcast = 0x150;
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v[I / kTokens]),
                                           kRowBroadcast + I % kTokens * kToken + C, 0xf, 0xf, true));
  }
  template <int I, int e>
  __device__ __forceinline__ float B() const { return at<I, e>(); }
  template <int I, int e>
  __device__ __forceinline__ float C() const { return at<I, E + e>(); }
};

// Token I's step of E states.
template <int I, int E, class T>
__device__ __forceinline__ void advance(const float (&A2)[E], const Coeffs<T, E>& bc, float2 v, float (&h)[E],
                                        float (&a)[E]) {
  each<E>([&](auto e_) {
    constexpr int e = decltype(e_)::value;
    a[e] = exp2_of(v.x * A2[e]);
    h[e] = fmaf(a[e], h[e], v.y * bc.template B<I, e>());
  });
}

// ---------------------------------------------------------------------------
// Forward: a wave has 16 channels, four lanes to each, and a lane four states (and every
// 16th four after them, NG in all). A lane reads B and C of its states, forms the step
// sizes of four of a batch's 16 tokens, which the channel's other lanes take from it, and
// ends with the outputs of these four. So waves neither wait for one another nor share
// memory, and one wave a SIMD, which is all that many calls have, is kept busy by its own
// four chains. (In fp32 and for N over 16 the compiler keeps a thread's eight inputs of the
// first launch in shared memory, 8 KiB a workgroup; no thread reads another's. 64 channels
// a wave, states over the waves, sums through shared memory with
// a barrier a batch: B8 T2048 H2048 N16 took 530 us for 1 wave a SIMD.)
// ---------------------------------------------------------------------------
constexpr int kFE = 4;                 // states of a lane
constexpr int kFParts = 4;             // lanes of a channel
constexpr int kFOwn = kL / kFParts;    // a lane's own tokens
constexpr int kFWaves = 4;             // of a workgroup, 64 channels together
constexpr int kFAhead = 4;             // tokens whose coefficients are under way

// Lane Q of each four's value.
template <int Q>
__device__ __forceinline__ float quad_take(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), Q * 0x55, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Of four sums over the four lanes, lane q's is the q-th.
__device__ __forceinline__ float quad_sums(float v0, float v1, float v2, float v3, int part) {
  const bool hi = part & 2, odd = part & 1;
  const float a = (hi ? v2 : v0) + dpp<0x4e>(hi ? v0 : v2);
  const float b = (hi ? v3 : v1) + dpp<0x4e>(hi ? v1 : v3);
  return (odd ? b : a) + dpp<0xb1>(odd ? a : b);
}

// How a lane finds its states among N: they are all there; all or none; any number.
constexpr int kAllThere = 0, kAllOrNone = 1, kSome = 2;

// B and C of a lane's E states, without a branch: one would stand between the loads of a
// token and the arithmetic of another.
template <class T, int E, int KIND, bool BOTH>
struct States {
  T b[KIND == kSome ? E : 1], c[KIND == kSome ? E : 1];
  Vec<T, E> vb, vc;
  __device__ __forceinline__ void load(const T* rowb, const T* rowc, int first, int N) {
    if constexpr (KIND == kSome) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        b[e] = lane_of(rowb, min(first + e, N - 1));
        if (BOTH) c[e] = lane_of(rowc, min(first + e, N - 1));
      }
    } else {
      const int at = KIND == kAllThere ? first : min(first, N - E);
      __builtin_memcpy(vb.w, &lane_of(rowb, at), sizeof(vb.w));
      if (BOTH) __builtin_memcpy(vc.w, &lane_of(rowc, at), sizeof(vc.w));
    }
  }
  __device__ __forceinline__ float B(int e, int n) const {
    if constexpr (KIND == kSome) return e < n ? (float)b[e] : 0.f;
    else return KIND == kAllThere || n > 0 ? vb.get(e) : 0.f;
  }
  __device__ __forceinline__ float C(int e, int n) const {
    if constexpr (KIND == kSome) return e < n ? (float)c[e] : 0.f;
    else return KIND == kAllThere || n > 0 ? vc.get(e) : 0.f;
  }
};

// STATE: the states that leave each chunk alone, each chunk from nothing.
template <class T, int NG, int KIND, bool STATE>
__global__ __launch_bounds__(64 * kFWaves) void ssm_fwd_kernel(SsmArgs p) {
  const Work w(p);
  const int part = w.lane % kFParts, hpg = p.H / p.G;
  const int local = (w.hb * kFWaves + w.wave) * 16 + w.lane / kFParts;
  const bool in = local < hpg;
  const int ch = w.g * hpg + (in ? local : 0);
  const long long HN = (long long)p.H * p.N, row = (long long)ch * p.N;
  auto first_of = [&](int r) { return (r * kFParts + part) * kFE; };  // of the lane's states
  // n states from the lane's r-th first, of a row of states; zero behind the last
  auto get = [&](const float* from, int r, float (&h)[kFE]) {
    const int n = p.N - first_of(r);
    Vec<float, kFE> v{};
    if (from != nullptr && in && n > 0) v = load_vec<float, kFE>(from + row + first_of(r), n);
#pragma unroll
    for (int e = 0; e < kFE; ++e) {
      h[e] = v.get(e);
      settle(h[e]);
    }
  };
  auto put = [&](float* to, int r, const float (&h)[kFE]) {
    const int n = p.N - first_of(r);
    Vec<float, kFE> v;
    v.put(h);
    if (in && n > 0) store_vec<float, kFE>(to + row + first_of(r), v, n);
  };
  float A2[NG][kFE], h[NG][kFE];
#pragma unroll
  for (int r = 0; r < NG; ++r) {
    get(p.A, r, A2[r]);
#pragma unroll
    for (int e = 0; e < kFE; ++e) A2[r][e] *= kLog2e;
    get(!STATE && p.chunks > 1 ? p.ends + w.chunk * HN : nullptr, r, h[r]);
  }
  float bias = p.dbias != nullptr ? p.dbias[ch] : 0.f, skip = p.D != nullptr ? p.D[ch] : 0.f;
  settle(bias);
  settle(skip);
  // the lane's own tokens from its first, of the batch at t; tokens behind the chunk's last
  // are it once more
  const T* px = static_cast<const T*>(p.x) + w.off(p, p.sxb, p.sxt) + ch;
  const T* pd = static_cast<const T*>(p.d) + w.off(p, p.sdb, p.sdt) + ch;
  const T* pz = p.z != nullptr ? static_cast<const T*>(p.z) + w.off(p, p.szb, p.szt) + ch : nullptr;
  struct Own {
    T x[kFOwn], d[kFOwn], z[kFOwn];
  };
  auto load = [&](int t, Own& o) {
    auto rows = [&](const T* base, long long st, T (&v)[kFOwn]) {
      if (t + kL <= w.c1) {
        const T* q = base + (t + part * kFOwn) * st;
#pragma unroll
        for (int j = 0; j < kFOwn; ++j, q += st) v[j] = *q;
      } else {
#pragma unroll
        for (int j = 0; j < kFOwn; ++j) v[j] = base[min(t + part * kFOwn + j, w.c1 - 1) * st];
      }
    };
    rows(px, p.sxt, o.x);
    rows(pd, p.sdt, o.d);
    if (!STATE && pz != nullptr) rows(pz, p.szt, o.z);
  };
  const T* pb = static_cast<const T*>(p.Bm) + w.off(p, p.sbb, p.sbt) + w.g * p.sbg;
  const T* pc = static_cast<const T*>(p.Cm) + w.off(p, p.scb, p.sct) + w.g * p.scg;
  Own own;
  load(w.c0, own);
  float sumd = 0.f;
  bool dropped = false;
  Seq seq{-1, 0, 0, 0};
  for (int t = w.c0; t < w.c1; t += kL) {
    Edges ed;
    ed.find(p.cu, p.B, p.T, (int)p.ntok, t, w.c1, seq);
    float dt[kFOwn], u[kFOwn];
#pragma unroll
    for (int j = 0; j < kFOwn; ++j) {
      dt[j] = (float)own.d[j] + bias;
      if (p.softplus) dt[j] = softplus(dt[j]);
      u[j] = dt[j] * (float)own.x[j];
      if (STATE && (ed.valid >> (part * kFOwn + j) & 1)) sumd += dt[j];
    }
    Own next = own;
    if (t + kL < w.c1) load(t + kL, next);
    if (!STATE && p.saved != nullptr && !(ed.start & 1)) {
#pragma unroll
      for (int r = 0; r < NG; ++r) put(p.saved + (w.b * p.tiles + (t - w.first) / kL) * HN, r, h[r]);
    }
    float y[kL];
    auto run = [&](auto edge_) {
      constexpr bool EDGE = decltype(edge_)::value;
      each<NG>([&](auto r_) {
        constexpr int r = decltype(r_)::value;
        const int first = first_of(r), n = p.N - first;
        States<T, kFE, KIND, !STATE> now[kFAhead], then[kFAhead];
        const T* rowb = pb + t * p.sbt;
        const T* rowc = pc + t * p.sct;
        auto coeffs = [&](int i, States<T, kFE, KIND, !STATE>& k) {
          if constexpr (EDGE) {
            const long long at = min(t + i, w.c1 - 1);
            k.load(pb + at * p.sbt, pc + at * p.sct, first, p.N);
          } else {
            k.load(rowb, rowc, first, p.N);
            rowb += p.sbt;
            rowc += p.sct;
          }
        };
#pragma unroll
        for (int j = 0; j < kFAhead; ++j) coeffs(j, now[j]);
        each<kL>([&](auto i_) {
          constexpr int i = decltype(i_)::value;
          if constexpr (i % kFAhead == 0 && i > 0) {
#pragma unroll
            for (int j = 0; j < kFAhead; ++j) now[j] = then[j];
          }
          if constexpr (i % kFAhead == 0 && i + kFAhead < kL) {
#pragma unroll
            for (int j = 0; j < kFAhead; ++j) coeffs(i + kFAhead + j, then[j]);
          }
          // otherwise all of a batch's loads go first, and their registers are not there
          if constexpr (i % kFAhead == 0) __builtin_amdgcn_sched_barrier(0);
          if (r == 0) y[i] = 0.f;
          if (EDGE && !(ed.valid >> i & 1)) return;
          if (EDGE && (ed.start >> i & 1)) {
            const float* from = nullptr;
            if (p.h0 != nullptr) at_state(p, t + i, [&](long long s) { from = p.h0 + s; });
            get(from, r, h[r]);
            if (i == 0 && !STATE && p.saved != nullptr)
              put(p.saved + (w.b * p.tiles + (t - w.first) / kL) * HN, r, h[r]);
          }
          const float di = quad_take<i / kFOwn>(dt[i % kFOwn]), ui = quad_take<i / kFOwn>(u[i % kFOwn]);
          const States<T, kFE, KIND, !STATE>& k = now[i % kFAhead];
          float part_y = 0.f;
#pragma unroll
          for (int e = 0; e < kFE; ++e) {
            h[r][e] = fmaf(exp2_of(di * A2[r][e]), h[r][e], ui * k.B(e, n));
            if (!STATE) part_y = e == 0 ? k.C(e, n) * h[r][e] : fmaf(k.C(e, n), h[r][e], part_y);
          }
          if (!STATE) y[i] = r == 0 ? part_y : y[i] + part_y;
          if (!STATE && EDGE && (ed.end >> i & 1)) at_state(p, t + i, [&](long long s) { put(p.hf + s, r, h[r]); });
        });
      });
    };
    if ((ed.start | ed.end) == 0 && ed.valid == kAll) run(std::false_type{});
    else run(std::true_type{});
    dropped = dropped || ed.start != 0 || ed.valid != kAll;
    if (!STATE) {
      T* out = static_cast<T*>(p.out) + (long long)(t + part * kFOwn) * p.H + ch;
#pragma unroll
      for (int j = 0; j < kFOwn; ++j, out += p.H) {
        float v = quad_sums(y[j], y[kFOwn + j], y[2 * kFOwn + j], y[3 * kFOwn + j], part);
        v = fmaf(skip, (float)own.x[j], v);
        if (pz != nullptr) {
          const float z = (float)own.z[j];
          v *= z * sigmoid(z);
        }
        const int i = part * kFOwn + j;
        if (in && t + i < w.c1) *out = (T)(ed.valid >> i & 1 ? v : 0.f);
      }
    }
    own = next;
  }
  if (STATE) {
#pragma unroll
    for (int r = 0; r < NG; ++r) put(p.ends + w.chunk * HN, r, h[r]);
    sumd += dpp<0xb1>(sumd);
    sumd += dpp<0x4e>(sumd);
    if (in && part == 0) p.sumd[w.chunk * p.H + ch] = sumd;
    if (w.g == 0 && w.hb == 0 && threadIdx.x == 0) p.drops[w.chunk] = dropped;
  }
}

// exp2(x) v + e. Where the exponential alone would leave the range its whole powers of two
// are applied last: a v of zero stays zero, a small one becomes what it is by definition.
__device__ __forceinline__ float joined(float x, float v, float e) {
  if (!(x > 126.f)) return fmaf(exp2_of(x), v, e);
  const float whole = rintf(x);
  return ldexpf(exp2_of(x - whole) * v, (int)fminf(whole, 1024.f)) + e;
}

// What enters each chunk, from what leaves the chunks before it, in their order (backward:
// after it, from the last).
template <bool BWD>
__global__ __launch_bounds__(256) void ssm_carry_kernel(SsmArgs p) {
  constexpr int kAhead = 8;
  const long long hn = (long long)p.H * p.N;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.lines * hn) return;
  const long long line = i / hn, at = i - line * hn;
  const int ch = (int)(at / p.N);
  const float A2 = p.A[at] * kLog2e;
  float carry = 0.f;
  for (int j0 = 0; j0 < p.chunks; j0 += kAhead) {
    float e[kAhead], d[kAhead];
    int lost[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = min(j0 + k, p.chunks - 1);
      const long long c = line * p.chunks + (BWD ? p.chunks - 1 - j : j);
      e[k] = p.ends[c * hn + at];
      d[k] = p.sumd[c * p.H + ch];
      lost[k] = p.drops[c];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (j0 + k >= p.chunks) break;
      const long long c = line * p.chunks + (BWD ? p.chunks - 1 - j0 - k : j0 + k);
      p.ends[c * hn + at] = carry;
      carry = lost[k] ? e[k] : joined(A2 * d[k], carry, e[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
constexpr int kBE = kSsmBwdStates;  // states of a wave
constexpr int kBMine = kL / kSsmWavesMax;

// A long sum that carries along what its last addition has lost (Kahan, Further Remarks on
// Reducing Truncation Errors, 1965): two roundings, however many terms. Of terms that are
// not finite it is what plain additions give.
struct Sum {
  float s = 0.f, over = 0.f;
  __device__ __forceinline__ void add(float v) {
    const float y = v - over, t = s + y;
    over = t - t == 0.f ? (t - s) - y : 0.f;
    s = t;
  }
};

// The sums over the 64 lanes of 64 values a lane, value l's in lane l. Each step halves the
// values: a lane keeps those whose bit is its own and adds what its partner has of them.
template <int HALF, int CTRL>
__device__ __forceinline__ void halve(float (&v)[64], bool upper) {
#pragma unroll
  for (int i = 0; i < HALF; ++i) {
    const float keep = upper ? v[i + HALF] : v[i], send = upper ? v[i] : v[i + HALF];
    v[i] = keep + dpp<CTRL>(send);
  }
}
__device__ __forceinline__ float sum_lanes(float (&v)[64], int lane) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 32]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 16]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  halve<8, 0x128>(v, lane & 8);  // lane ^ 8: a rotation by 8 in its row
  halve<4, 0x141>(v, lane & 4);  // 7 - lane in its half of a row
  halve<2, 0x4e>(v, lane & 2);   // lane ^ 2
  halve<1, 0xb1>(v, lane & 1);   // lane ^ 1
  return v[0];
}

// Reverse of the forward's STATE: the gradient that leaves each chunk at its front.
template <class T, int NG>
__global__ __launch_bounds__(64 * kSsmWavesMax) __attribute__((amdgpu_waves_per_eu(NG == 4 ? 2 : 4))) void
ssm_bwd_state_kernel(SsmArgs p) {
  __shared__ float2 dd[2][kL][64];  // step size, dy
  __shared__ float sums[kSsmWavesMax][64];
  constexpr int waves = kSsmWavesMax;
  const int pairs = (p.N + kBE - 1) / kBE;
  const Work w(p);
  float A2[NG][kBE], g[NG][kBE];
#pragma unroll
  for (int r = 0; r < NG; ++r) {
#pragma unroll
    for (int e = 0; e < kBE; ++e) g[r][e] = 0.f;
    read_rates<kBE>(p, w, r * waves + w.wave, A2[r]);
  }
  float bias = p.dbias != nullptr && w.in ? p.dbias[w.ch] : 0.f;
  settle(bias);
  float sumd = 0.f;
  bool dropped = false;
  Inputs<T, kBMine> cur, next;
  Coeffs<T, kBE> bc[NG], bc_next[NG];
  auto load = [&](int t, Inputs<T, kBMine>& v, Coeffs<T, kBE> (&c)[NG]) {
    v.template load<true>(p, w, waves, t);
#pragma unroll
    for (int r = 0; r < NG; ++r) c[r].load(p, w, r * waves + w.wave, t);
  };
  const int last = w.c0 + (w.c1 - 1 - w.c0) / kL * kL;
  load(last, cur, bc);
  Seq seq{-1, 0, 0, 0};
  int buf = 0;
  for (int t = last; t >= w.c0; t -= kL, buf ^= 1) {
    Edges ed;
    ed.find(p.cu, p.B, p.T, (int)p.ntok, t, w.c1, seq);
    if (t > w.c0) load(t - kL, next, bc_next);
#pragma unroll
    for (int j = 0; j < kBMine; ++j) {
      const int i = w.wave + j * waves;
      float dt = (float)cur.d[j] + bias;
      if (p.softplus) dt = softplus(dt);
      float dy = (float)cur.go[j];
      if (p.z != nullptr) dy *= (float)cur.z[j] * sigmoid((float)cur.z[j]);
      const bool ok = ed.valid >> i & 1;
      dd[buf][i][w.lane] = make_float2(ok ? dt : 0.f, ok ? dy : 0.f);
      sumd += ok ? dt : 0.f;
    }
    __syncthreads();
    for (unsigned rest = ed.valid, seg; rest != 0; rest &= ~seg) {
      seg = ed.last(rest);
      float2 v[kL];
#pragma unroll
      for (int i = 0; i < kL; ++i) v[i] = dd[buf][i][w.lane];
      if (seg != kAll) {
#pragma unroll
        for (int i = 0; i < kL; ++i)
          if (!(seg >> i & 1)) v[i] = make_float2(0.f, 0.f);
      }
      each<NG>([&](auto r_) {
        constexpr int r = decltype(r_)::value;
        const int q = r * waves + w.wave;
        if (q >= pairs) return;
        if (seg & ed.end) read_states<kBE>(p, w, q, p.gh, t + highest(seg), g[r]);
        bc[r].arrive(p, w, q, seg);
        back([&](auto i_) {
          constexpr int i = decltype(i_)::value;
          each<kBE>([&](auto e_) {
            constexpr int e = decltype(e_)::value;
            g[r][e] = exp2_of(v[i].x * A2[r][e]) * fmaf(bc[r].template C<i, e>(), v[i].y, g[r][e]);
          });
        });
        if (seg & ed.start) {
#pragma unroll
          for (int e = 0; e < kBE; ++e) g[r][e] = 0.f;
        }
      });
    }
    dropped = dropped || ed.start != 0 || (t + kL <= w.c1 && ed.valid != kAll);
    cur = next;
#pragma unroll
    for (int r = 0; r < NG; ++r) bc[r] = bc_next[r];
  }
#pragma unroll
  for (int r = 0; r < NG; ++r)
    states<kBE>(p, w, r * waves + w.wave,
                [&](int e, long long at) { p.ends[w.chunk * p.N * p.H + at] = g[r][e]; });
  sums[w.wave][w.lane] = sumd;
  __syncthreads();
  if (w.wave == 0 && w.in) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < waves; ++k) s += sums[k][w.lane];
    p.sumd[w.chunk * p.H + w.ch] = s;
  }
  if (w.g == 0 && w.hb == 0 && threadIdx.x == 0) p.drops[w.chunk] = dropped;
}

template <class T, int NG>
__global__ __launch_bounds__(64 * kSsmWavesMax) void ssm_bwd_kernel(SsmArgs p) {
  extern __shared__ float shared[];
  constexpr int waves = kSsmWavesMax;
  const int pairs = (p.N + kBE - 1) / kBE, active = pairs < waves ? pairs : waves;
  float2* du = reinterpret_cast<float2*>(shared);            // [kL][64]: step size, times x
  float* dys = shared + kL * 64 * 2;                         // [kL][64]
  float2* s12 = reinterpret_cast<float2*>(dys + kL * 64);    // [waves][kL][64]
  float* s3 = dys + kL * 64 + waves * kL * 64 * 2;           // [waves][kL][64], with z only
  const Work w(p);
  const long long HN = (long long)p.H * p.N;
  float A2[NG][kBE], g[NG][kBE];
  Sum dA[NG][kBE];
#pragma unroll
  for (int r = 0; r < NG; ++r) {
    const int q = r * waves + w.wave;
#pragma unroll
    for (int e = 0; e < kBE; ++e) g[r][e] = 0.f;
    read_rates<kBE>(p, w, q, A2[r]);
    if (p.chunks > 1)
      states<kBE>(p, w, q, [&](int e, long long at) { g[r][e] = p.ends[w.chunk * HN + at]; });
#pragma unroll
    for (int e = 0; e < kBE; ++e) settle(g[r][e]);
  }
  float bias = p.dbias != nullptr && w.in ? p.dbias[w.ch] : 0.f;
  float skip = p.D != nullptr && w.in ? p.D[w.ch] : 0.f;
  settle(bias);
  settle(skip);
  Sum dD, dbias;
  const bool gated = p.z != nullptr;
  const int last = w.c0 + (w.c1 - 1 - w.c0) / kL * kL;
  Inputs<T, kBMine> in, next;
  float hin[NG][kBE], hnext[NG][kBE];
  Coeffs<T, kBE> bc[NG], bc_next[NG];
  auto load = [&](int t, Inputs<T, kBMine>& v, float (&h)[NG][kBE], Coeffs<T, kBE> (&c)[NG]) {
    v.template load<true>(p, w, waves, t);
#pragma unroll
    for (int r = 0; r < NG; ++r) c[r].load(p, w, r * waves + w.wave, t);
    const float* from = p.saved + (w.b * p.tiles + (t - w.first) / kL) * HN;
    const int ch = w.in ? w.ch : 0;
#pragma unroll
    for (int r = 0; r < NG; ++r)
#pragma unroll
      for (int e = 0; e < kBE; ++e)
        h[r][e] = from[(long long)ch * p.N + min((r * waves + w.wave) * kBE + e, p.N - 1)];
  };
  load(last, in, hin, bc);
  if (w.wave >= active)
    for (int i = 0; i < kL; ++i) {
      s12[(w.wave * kL + i) * 64 + w.lane] = make_float2(0.f, 0.f);
      if (gated) s3[(w.wave * kL + i) * 64 + w.lane] = 0.f;
    }
  Seq seq{-1, 0, 0, 0};
  for (int t = last; t >= w.c0; t -= kL) {
    Edges ed;
    ed.find(p.cu, p.B, p.T, (int)p.ntok, t, w.c1, seq);
    if (t > w.c0) load(t - kL, next, hnext, bc_next);
#pragma unroll
    for (int j = 0; j < kBMine; ++j) {
      const int i = w.wave + j * waves;
      float dt = (float)in.d[j] + bias;
      if (p.softplus) dt = softplus(dt);
      float dy = (float)in.go[j];
      if (gated) dy *= (float)in.z[j] * sigmoid((float)in.z[j]);
      // lanes without a channel give nothing to the sums over channels
      const bool ok = w.in && (ed.valid >> i & 1);
      du[i * 64 + w.lane] = make_float2(ok ? dt : 0.f, ok ? dt * (float)in.x[j] : 0.f);
      dys[i * 64 + w.lane] = ok ? dy : 0.f;
    }
    __syncthreads();
    // sequence by sequence, from the last
    for (unsigned rest = w.wave < active ? ed.valid : 0u, seg; rest != 0; rest &= ~seg) {
      seg = ed.last(rest);
      float2 v[kL];
      float dy[kL];
#pragma unroll
      for (int i = 0; i < kL; ++i) {
        v[i] = du[i * 64 + w.lane];
        dy[i] = dys[i * 64 + w.lane];
      }
      if (seg != kAll) {
#pragma unroll
        for (int i = 0; i < kL; ++i)
          if (!(seg >> i & 1)) {
            v[i] = make_float2(0.f, 0.f);
            dy[i] = 0.f;
          }
      }
      each<NG>([&](auto r_) {
        constexpr int r = decltype(r_)::value;
        const int q = r * waves + w.wave;
        if (NG > 1 && q >= pairs) return;
        bc[r].arrive(p, w, q, seg);
        // the batch's decays and the states before its tokens once more; a lane without a
        // channel has read another group's, and its part in the sums over channels has to
        // be zero whatever they are
        float a[kL][kBE], hp[kL][kBE], h[kBE];
#pragma unroll
        for (int e = 0; e < kBE; ++e) h[e] = w.in ? hin[r][e] : 0.f;
        if (seg & ed.start & ~1u) read_states<kBE>(p, w, q, p.h0, t + lowest(seg), h);
        each<kL>([&](auto i_) {
          constexpr int i = decltype(i_)::value;
#pragma unroll
          for (int e = 0; e < kBE; ++e) hp[i][e] = h[e];
          advance<i, kBE>(A2[r], bc[r], v[i], h, a[i]);
        });
        if (seg & ed.end) read_states<kBE>(p, w, q, p.gh, t + highest(seg), g[r]);
        float sums[64], da[kBE] = {};
        back([&](auto i_) {
          constexpr int i = decltype(i_)::value;
          float s1 = 0.f, s2 = 0.f, y = 0.f;
          each<kBE>([&](auto e_) {
            constexpr int e = decltype(e_)::value;
            const float B = bc[r].template B<i, e>(), C = bc[r].template C<i, e>();
            const float ht = i + 1 < kL ? hp[i + 1 < kL ? i + 1 : 0][e] : h[e];
            const float d = fmaf(C, dy[i], g[r][e]);
            const float ga = a[i][e] * d;
            const float k = ga * hp[i][e];
            s1 = fmaf(B, d, s1);
            s2 = fmaf(A2[r][e], k, s2);
            y = fmaf(C, ht, y);
            da[e] = fmaf(v[i].x, k, da[e]);
            sums[i * 2 * kBE + e] = d * v[i].y;
            sums[i * 2 * kBE + kBE + e] = dy[i] * ht;
            g[r][e] = ga;
          });
          if (seg == kAll || (seg >> i & 1)) {
            const int at = (w.wave * kL + i) * 64 + w.lane;
            if (r == 0) {
              s12[at] = make_float2(s1, s2);
              if (gated) s3[at] = y;
            } else {
              s12[at] = make_float2(s12[at].x + s1, s12[at].y + s2);
              if (gated) s3[at] += y;
            }
          }
        });
#pragma unroll
        for (int e = 0; e < kBE; ++e) dA[r][e].add(da[e]);
        if (seg & ed.start) {
          if (p.gs != nullptr)
            at_state(p, t + lowest(seg), [&](long long s) {
              states<kBE>(p, w, q, [&](int e, long long at) { p.gs[s + at] = g[r][e]; });
            });
#pragma unroll
          for (int e = 0; e < kBE; ++e) g[r][e] = 0.f;
        }
        if (p.part_bc != nullptr) {
          const float s = sum_lanes(sums, w.lane);
          const long long all = (long long)p.G * pairs * p.ntok,
                          plane = (w.g * (long long)pairs + q) * p.ntok + t;
          const unsigned tok = w.lane / (2 * kBE);
          if (seg >> tok & 1) lane_of(p.part_bc + (w.hb * all + plane) * (2 * kBE), w.lane) = s;
        }
      });
    }
    if (p.part_bc != nullptr && ed.valid != kAll && w.wave < active) {
      // tokens outside the sequences
      const long long all = (long long)p.G * pairs * p.ntok;
      const int tok = w.lane / (2 * kBE);
      for (int q = w.wave; q < pairs; q += waves)
        if (t + tok < w.c1 && !(ed.valid >> tok & 1))
          p.part_bc[(w.hb * all + (w.g * (long long)pairs + q) * p.ntok + t) * (2 * kBE) + w.lane] = 0.f;
    }
    __syncthreads();
    float sum_d = 0.f, sum_b = 0.f;
#pragma unroll
    for (int j = 0; j < kBMine; ++j) {
      const int i = w.wave + j * waves;
      if (t + i >= w.c1 || !w.in) continue;
      const long long at = (long long)(t + i) * p.H;
      float s1 = 0.f, s2 = 0.f, y = 0.f;
#pragma unroll
      for (int k = 0; k < waves; ++k) {
        const float2 q = s12[(k * kL + i) * 64 + w.lane];
        s1 += q.x;
        s2 += q.y;
      }
      if (gated) {
#pragma unroll
        for (int k = 0; k < waves; ++k) y += s3[(k * kL + i) * 64 + w.lane];
      }
      const bool ok = ed.valid >> i & 1;
      const float x = (float)in.x[j], dy = dys[i * 64 + w.lane], dt = du[i * 64 + w.lane].x;
      // s2 holds A in units of log2(e)
      float gd = fmaf(x, s1, s2 * (1.f / kLog2e));
      if (p.softplus) gd *= sigmoid((float)in.d[j] + bias);
      const float gx = fmaf(dt, s1, skip * dy);
      if (ok) {
        sum_d = fmaf(dy, x, sum_d);
        sum_b += gd;
      }
      if (p.gx != nullptr) lane_of(static_cast<T*>(p.gx) + at, w.ch) = (T)(ok ? gx : 0.f);
      if (p.gd != nullptr) lane_of(static_cast<T*>(p.gd) + at, w.ch) = (T)(ok ? gd : 0.f);
      if (p.gz != nullptr) {
        const float z = (float)in.z[j], sg = sigmoid(z);
        const float gz = (float)in.go[j] * fmaf(skip, x, y) * sg * fmaf(z, 1.f - sg, 1.f);
        lane_of(static_cast<T*>(p.gz) + at, w.ch) = (T)(ok ? gz : 0.f);
      }
    }
    dD.add(sum_d);
    dbias.add(sum_b);
    in = next;
#pragma unroll
    for (int r = 0; r < NG; ++r) {
#pragma unroll
      for (int e = 0; e < kBE; ++e) hin[r][e] = hnext[r][e];
      bc[r] = bc_next[r];
    }
    __syncthreads();
  }
  if (p.part_a != nullptr) {
#pragma unroll
    for (int r = 0; r < NG; ++r)
      states<kBE>(p, w, r * waves + w.wave, [&](int e, long long at) { p.part_a[w.chunk * HN + at] = dA[r][e].s; });
  }
  if (p.part_h != nullptr) {
    shared[w.wave * 64 + w.lane] = dD.s;
    shared[(waves + w.wave) * 64 + w.lane] = dbias.s;
    __syncthreads();
    if (w.wave < 2 && w.in) {
      float s = 0.f;
      for (int k = 0; k < waves; ++k) s += shared[(w.wave * waves + k) * 64 + w.lane];
      p.part_h[(w.chunk * 2 + w.wave) * p.H + w.ch] = s;
    }
  }
}

// dB and dC from the blocks of channels.
template <class T>
__global__ __launch_bounds__(256) void ssm_sum_bc_kernel(SsmArgs p) {
  const int pairs = (p.N + kBE - 1) / kBE;
  const long long per = p.ntok * (2 * kBE), total = (long long)p.G * pairs * per;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float s = 0.f;
  for (int b = 0; b < p.hblocks; ++b) s += p.part_bc[b * total + i];
  const long long gq = i / per, rest = i - gq * per;
  const long long t = rest / (2 * kBE);
  const int g = (int)(gq / pairs), c = (int)(rest % (2 * kBE));
  const int n = (int)(gq - (long long)g * pairs) * kBE + c % kBE;
  if (n >= p.N) return;
  void* to = c < kBE ? p.gB : p.gC;
  if (to != nullptr) static_cast<T*>(to)[(t * p.G + g) * p.N + n] = (T)s;
}

// dA, dD and the bias's from the chunks, in kParts interleaved parts.
__global__ __launch_bounds__(256) void ssm_sum_par_kernel(SsmArgs p) {
  constexpr int kCols = 32, kParts = 256 / kCols;
  __shared__ float sums[kParts][kCols];
  const long long hn = (long long)p.H * p.N, cols = hn + 2 * p.H, items = p.lines * p.chunks;
  const long long col = (long long)blockIdx.x * kCols + threadIdx.x % kCols;
  const int part = threadIdx.x / kCols;
  const float* from = col < hn ? p.part_a + col : p.part_h + (col - hn);
  const long long stride = col < hn ? hn : 2 * p.H;
  Sum of;
  if (col < cols)
    for (long long i = part; i < items; i += kParts) of.add(from[i * stride]);
  sums[part][threadIdx.x % kCols] = of.s;
  __syncthreads();
  if (part > 0 || col >= cols) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) s += sums[i][threadIdx.x];
  if (col < hn) {
    if (p.gA != nullptr) p.gA[col] = s;
  } else if (col < hn + p.H) {
    if (p.gD != nullptr) p.gD[col - hn] = s;
  } else if (p.gbias != nullptr) {
    p.gbias[col - hn - p.H] = s;
  }
}

// ---------------------------------------------------------------------------
// One token of each stream: `lanes` threads to a channel, four states to each (more in
// rounds). The states' bytes bound it: each is read and written once.
// ---------------------------------------------------------------------------
constexpr int kStepThreads = 256;
constexpr int kSE = 4;  // states of a thread

template <class T>
__global__ __launch_bounds__(kStepThreads) void ssm_step_kernel(SsmStepArgs p, int lanes) {
  const int row = blockIdx.y;
  const int lane = threadIdx.x & (lanes - 1);
  const int ch = blockIdx.x * (kStepThreads / lanes) + threadIdx.x / lanes;
  const bool in = ch < p.H;
  const int slot = p.slots != nullptr ? p.slots[row] : row;
  const bool live = slot >= 0 && slot < p.P;
  const int n0 = lane * kSE, n = p.N - n0;
  const int g = in ? ch / (p.H / p.G) : 0;
  float* state = p.state + slot * p.ssp + (long long)ch * p.N + n0;
  Vec<float, kSE> h{}, A{};
  float bias = 0.f, skip = 0.f;
  Vec<T, kSE> bm{}, cm{};
  T x{}, d{}, z{};
  const auto load = [&](int r) {
    x = static_cast<const T*>(p.x)[r * p.sx + ch];
    d = static_cast<const T*>(p.d)[r * p.sd + ch];
    if (p.z != nullptr) z = static_cast<const T*>(p.z)[r * p.sz + ch];
    if (n > 0) {
      bm = load_vec<T, kSE>(static_cast<const T*>(p.Bm) + r * p.sbb + g * p.sbg + n0, n);
      cm = load_vec<T, kSE>(static_cast<const T*>(p.Cm) + r * p.scb + g * p.scg + n0, n);
    }
  };
  if (in && live) {
    if (n > 0) {
      h = load_vec<float, kSE>(state, n);
      A = load_vec<float, kSE>(p.A + (long long)ch * p.N + n0, n);
    }
    load(row);
    if (p.dbias != nullptr) bias = p.dbias[ch];
    if (p.D != nullptr) skip = p.D[ch];
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
      if (in && lane == 0) out[(long long)row * p.H] = (T)(slot < 0 ? 0.f : __builtin_nanf(""));
      return;
    }
    if (earlier) return;
  }
  float f[kSE];
#pragma unroll
  for (int e = 0; e < kSE; ++e) f[e] = h.get(e);
  auto step = [&](int r) {
    const float xf = (float)x;
    float y = 0.f, dt = (float)d + bias;
    if (p.softplus) dt = softplus(dt);
#pragma unroll
    for (int e = 0; e < kSE; ++e)
      if (e < n) {
        f[e] = fmaf(exp2_of(dt * (A.get(e) * kLog2e)), f[e], dt * xf * bm.get(e));
        y = fmaf(cm.get(e), f[e], y);
      }
    for (int o = lanes / 2; o > 0; o /= 2) y += __shfl_xor(y, o);
    if (in && lane == 0) {
      y = fmaf(skip, xf, y);
      if (p.z != nullptr) y *= (float)z * sigmoid((float)z);
      out[(long long)r * p.H] = (T)y;
    }
  };
  step(row);
  if (more)
    for (int r = row + 1; r < p.B; ++r) {
      if (p.slots[r] != slot) continue;
      if (in) load(r);
      step(r);
    }
  if (in && n > 0) {
    h.put(f);
    store_vec<float, kSE>(state, h, n);
  }
}

template <class F>
hipError_t with_type(int type, F&& f) {
  if (type == LTC_F32) return f(float{});
  if (type == LTC_BF16) return f(__bf16{});
  return f(_Float16{});
}

// Calls f with the rounds that a wave takes, 16 states each.
template <class F>
hipError_t with_rounds(int N, F&& f) {
  if (N <= 16) return f(std::integral_constant<int, 1>{});
  if (N <= 32) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}
// And with how the lanes find their states.
template <class F>
hipError_t with_states(int N, F&& f) {
  return with_rounds(N, [&](auto ng) {
    if (N % (16 * decltype(ng)::value) == 0) return f(ng, std::integral_constant<int, kAllThere>{});
    if (N % 4 == 0) return f(ng, std::integral_constant<int, kAllOrNone>{});
    return f(ng, std::integral_constant<int, kSome>{});
  });
}

hipError_t launch_empty(const SsmArgs& a, const float* src, float* dst, hipStream_t s) {
  if (dst == nullptr) return hipSuccess;
  const long long blocks = ((long long)a.B * a.H * a.N + 255) / 256;
  LTC_LAUNCH(ssm_empty_kernel, dim3((unsigned)(blocks > 4096 ? 4096 : blocks)), dim3(256), 0, s, a, src, dst);
  return hipGetLastError();
}

unsigned carry_groups(const SsmArgs& a) { return (unsigned)((a.lines * a.H * a.N + 255) / 256); }

}  // namespace

// Workgroups of 64 channels. Where they are too few for the chip, sequences are cut.
void ssm_plan(SsmArgs* a, bool packed, bool bwd) {
  a->hblocks = (a->H / a->G + 63) / 64;
  a->lines = packed ? 1 : a->B;
  a->tiles = (a->T + kL - 1) / kL;
  const long long base = a->lines * a->G * a->hblocks, want = bwd ? 256 : 1024;
  long long chunks = 1;
  if (base > 0 && base < 256) chunks = (want + base - 1) / base;
  const long long most = (a->T + 4 * kL - 1) / (4 * kL);
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  long long len = (a->T + chunks - 1) / chunks;
  len = (len + kL - 1) / kL * kL;
  a->len = (int)(len < kL ? kL : len);
  a->chunks = a->T > 0 ? (int)((a->T + a->len - 1) / a->len) : 0;
}

hipError_t launch_ssm_fwd(int type, const SsmArgs& a, hipStream_t s) {
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const bool ends = a.B > 0 && (a.cu != nullptr || a.ntok == 0);
    hipError_t e = launch_empty(a, a.h0, ends ? a.hf : nullptr, s);
    if (e != hipSuccess || a.ntok == 0) return e;
    return with_states(a.N, [&](auto ng, auto kind) {
      constexpr int NG = decltype(ng)::value, KIND = decltype(kind)::value;
      const dim3 grid((unsigned)(a.lines * a.chunks * a.G * a.hblocks)), block(64 * kFWaves);
      if (a.chunks > 1) {
        LTC_LAUNCH((ssm_fwd_kernel<T, NG, KIND, true>), grid, block, 0, s, a);
        LTC_LAUNCH((ssm_carry_kernel<false>), dim3(carry_groups(a)), dim3(256), 0, s, a);
      }
      LTC_LAUNCH((ssm_fwd_kernel<T, NG, KIND, false>), grid, block, 0, s, a);
      return hipGetLastError();
    });
  });
}

hipError_t launch_ssm_bwd(int type, const SsmArgs& a, hipStream_t s) {
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const bool ends = a.gs != nullptr && a.B > 0 && (a.cu != nullptr || a.ntok == 0);
    hipError_t e = launch_empty(a, a.gh, ends ? a.gs : nullptr, s);
    if (e != hipSuccess) return e;
    if (a.ntok > 0) {
      e = with_rounds(a.N, [&](auto ng) {
        constexpr int NG = decltype(ng)::value;
          const dim3 grid((unsigned)(a.lines * a.chunks * a.G * a.hblocks)), block(64 * kSsmWavesMax);
        if (a.chunks > 1) {
          LTC_LAUNCH((ssm_bwd_state_kernel<T, NG>), grid, block, 0, s, a);
          LTC_LAUNCH((ssm_carry_kernel<true>), dim3(carry_groups(a)), dim3(256), 0, s, a);
        }
        const size_t lds = (kL * 64 * 3 + kSsmWavesMax * kL * 64 * (a.z != nullptr ? 3 : 2)) * sizeof(float);
        LTC_LAUNCH((ssm_bwd_kernel<T, NG>), grid, block, lds, s, a);
        return hipGetLastError();
      });
      if (e != hipSuccess) return e;
      if (a.part_bc != nullptr) {
        const long long n = a.ntok * 2 * kBE * a.G * ((a.N + kBE - 1) / kBE);
        LTC_LAUNCH((ssm_sum_bc_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
      }
    }
    if (a.gA != nullptr || a.gD != nullptr || a.gbias != nullptr) {
      const long long cols = (long long)a.H * a.N + 2 * a.H;
      LTC_LAUNCH(ssm_sum_par_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(256), 0, s, a);
    }
    return hipGetLastError();
  });
}

hipError_t launch_ssm_step(int type, const SsmStepArgs& a, hipStream_t s) {
  if (a.B == 0) return hipSuccess;
  int lanes = 1;
  while (lanes * kSE < a.N) lanes *= 2;
  const int per = kStepThreads / lanes;
  const dim3 grid((a.H + per - 1) / per, a.B);
  return with_type(type, [&](auto t) {
    LTC_LAUNCH((ssm_step_kernel<decltype(t)>), grid, dim3(kStepThreads), 0, s, a, lanes);
    return hipGetLastError();
  });
}

}  // namespace ltc
