// Selective state space scan, for gfx950. Of every channel c and state n:
//   D_t = delta_t (+ bias), or softplus of it      a = exp(D_t A[c,n])
//   h_t = a h_{t-1} + D_t B_t[n] x_t               y_t = sum_n C_t[n] h_t + skip x_t
//   out_t = y_t, or y_t silu(z_t)
// Backward, with dy = dout or dout silu(z) and d_t = C_t dy_t + a_{t+1} d_{t+1}:
//   dL/dB_t[n] = sum_c d D x      dL/dC_t[n] = sum_c dy h      s1 = sum_n d B
//   dL/dx = D s1 + skip dy        dL/dD = x s1 + sum_n A a h_{t-1} d
//   dL/dA = sum_t D a h_{t-1} d
//
// Arithmetic bounds it: forward a product, an exponential (four times a product's time), a
// product and two multiply-adds a state; backward these once more and about twelve. A
// workgroup has 64 channels, one to a lane, and walks a chunk of the time axis in batches
// of 16 tokens; its waves share the states, four to a wave. So B_t and C_t, the same for
// all lanes, come through the scalar unit, from a copy that a small launch lays out; step
// sizes are formed once, by one wave each, and handed round in shared memory; and so are
// the waves' parts of the sums over states. The sums over channels, for dB and dC, are
// formed by halving: 64 sums over 64 lanes take 63 exchanges instead of 384.
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
constexpr int kE = 4;  // states of a wave

typedef float F8 __attribute__((ext_vector_type(8)));
typedef const F8 __attribute__((address_space(4))) * ScalarF8;

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
  const float l = f == 0.f ? e : __logf(w) * (e * __builtin_amdgcn_rcpf(f));
  return fmaxf(v, 0.f) + l;
}

template <class T>
__device__ __forceinline__ float value(const T* p) {
  return (float)*p;
}

// ---------------------------------------------------------------------------
// Preparation: B and C of four states and a token as eight floats, zero outside the
// sequences and behind the last state; and the ends of sequences without tokens.
// ---------------------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(256) void ssm_prep_kernel(SsmArgs p, const float* src, float* dst) {
  const long long per = (long long)p.G * p.quads, total = p.ntok * per;
  const long long i0 = (long long)blockIdx.x * 256 + threadIdx.x, step = (long long)gridDim.x * 256;
  for (long long i = i0; i < total; i += step) {
    const int t = (int)(i / per), r = (int)(i - t * per);
    const int g = r / p.quads, q = r - g * p.quads;
    const Seq s = seq_of(p.cu, p.B, p.T, (int)p.ntok, t, 0, 0);
    float f[8] = {};
    if (s.s >= 0) {
      const T* b = static_cast<const T*>(p.Bm) + g * p.sbg;
      const T* c = static_cast<const T*>(p.Cm) + g * p.scg;
      if (p.cu == nullptr) {
        b += s.s * p.sbb + (t - s.lo) * p.sbt;
        c += s.s * p.scb + (t - s.lo) * p.sct;
      } else {
        b += t * p.sbt;
        c += t * p.sct;
      }
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (q * kE + e < p.N) {
          f[e] = value(b + q * kE + e);
          f[kE + e] = value(c + q * kE + e);
        }
    }
    float* to = p.bc + ((g * (long long)p.quads + q) * p.ntok + t) * 8;
    __builtin_memcpy(to, f, sizeof(f));
  }
  if (dst != nullptr) {
    const long long hn = (long long)p.H * p.N;
    for (long long i = i0; i < p.B * hn; i += step) {
      int lo = 0, hi = 0;
      if (p.ntok > 0) span_of(p.cu, p.T, (int)p.ntok, (int)(i / hn), lo, hi);
      if (lo == hi) dst[i] = src != nullptr ? src[i] : 0.f;
    }
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
    const long long first = b * p.T + (chunk - b * p.chunks) * (long long)p.len;
    const long long last = b * p.T + p.T;
    c0 = (int)first;
    c1 = (int)(first + p.len < last ? first + p.len : last);
    const int hpg = p.H / p.G;
    in = hb * 64 + lane < hpg;
    ch = g * hpg + hb * 64 + lane;
  }
  // Element of token t of a tensor of strides sb, st, from which the lane's channel counts.
  __device__ __forceinline__ long long off(const SsmArgs& p, long long sb, long long st) const {
    return p.cu == nullptr ? b * (sb - p.T * st) : 0;
  }
};

// Which of a batch's tokens begin a sequence, end one, and lie in one.
struct Edges {
  unsigned start, end, valid;
  __device__ __forceinline__ bool none() const { return (start | end) == 0 && valid == (1u << kL) - 1; }
};
__device__ __forceinline__ Edges edges_of(const SsmArgs& p, int t, int c1) {
  Edges e{0, 0, 0};
  const int n = c1 - t < kL ? c1 - t : kL;
  int i = 0;
  while (i < n) {
    const Seq q = seq_of(p.cu, p.B, p.T, (int)p.ntok, t + i, 0, 0);
    const int m = q.hi - t < n ? q.hi - t : n;
    if (q.s >= 0) {
      if (q.lo == t + i) e.start |= 1u << i;
      if (q.hi - t <= n) e.end |= 1u << (q.hi - t - 1);
      e.valid |= ((1u << m) - 1) & ~((1u << i) - 1);
    }
    i = m;
  }
  return e;
}
__device__ __forceinline__ int seq_at(const SsmArgs& p, int t) {
  return seq_of(p.cu, p.B, p.T, (int)p.ntok, t, 0, 0).s;
}

// A wave's tokens of a batch: wave, wave + waves, ...; at most kMine.
constexpr int kMine = kL / kSsmWavesMin;

// The four states of quad q of a lane's channel in (rows,H,N).
template <class F>
__device__ __forceinline__ void states(const SsmArgs& p, const Work& w, int q, F&& f) {
#pragma unroll
  for (int e = 0; e < kE; ++e)
    if (w.in && q * kE + e < p.N) f(e, (long long)w.ch * p.N + q * kE + e);
}
// In (rows,N,H), where a wave's lanes lie side by side.
template <class F>
__device__ __forceinline__ void planes(const SsmArgs& p, const Work& w, int q, F&& f) {
#pragma unroll
  for (int e = 0; e < kE; ++e)
    if (w.in && q * kE + e < p.N) f(e, (long long)(q * kE + e) * p.H + w.ch);
}

template <class T>
struct Inputs {
  float x[kMine], d[kMine], z[kMine], go[kMine];
  // Of the batch at t; zero where there is no token.
  template <bool BWD>
  __device__ __forceinline__ void load(const SsmArgs& p, const Work& w, int t) {
    const T* px = static_cast<const T*>(p.x) + w.off(p, p.sxb, p.sxt) + w.ch;
    const T* pd = static_cast<const T*>(p.d) + w.off(p, p.sdb, p.sdt) + w.ch;
    const T* pz = static_cast<const T*>(p.z) + w.off(p, p.szb, p.szt) + w.ch;
    const T* pg = static_cast<const T*>(p.go) + (BWD ? w.off(p, p.sob, p.sot) : 0) + w.ch;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = w.wave + j * p.waves;
      const long long u = t + i;
      const bool there = i < kL && u < w.c1 && w.in;
      x[j] = there ? value(px + u * p.sxt) : 0.f;
      d[j] = there ? value(pd + u * p.sdt) : 0.f;
      z[j] = there && p.z != nullptr ? value(pz + u * p.szt) : 0.f;
      if (BWD) go[j] = there && p.go != nullptr ? value(pg + u * p.sot) : 0.f;
    }
  }
};

// Of a wave's four states and a token: the decays, B and C.
template <bool PAD>
__device__ __forceinline__ void quad_step(const float (&A2)[kE], F8 bc, float dt, float u, int ne, float (&h)[kE],
                                          float (&a)[kE]) {
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    // a state behind the last stays 0, whatever the token
    const bool no = PAD && e >= ne;
    a[e] = exp2_of((no ? 0.f : dt) * A2[e]);
    h[e] = fmaf(a[e], h[e], (no ? 0.f : u) * bc[e]);
  }
}

__device__ __forceinline__ F8 bc_at(const float* p) {
  return *(ScalarF8)(reinterpret_cast<uintptr_t>(p));
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
// STATE: the states that leave each chunk alone, each chunk from nothing.
template <class T, int NG, bool PAD, bool STATE>
__global__ __launch_bounds__(64 * kSsmWavesMax) void ssm_fwd_kernel(SsmArgs p) {
  extern __shared__ float shared[];
  float2* du = reinterpret_cast<float2*>(shared);       // [2][kL][64]: step size, times x
  float* ys = shared + 2 * kL * 64 * 2;                 // [2][waves][kL][64]
  const Work w(p);
  const int waves = p.waves, active = p.quads < waves ? p.quads : waves;
  float A2[NG][kE], h[NG][kE];
  const float* bcq[NG];
  int ne[NG];
#pragma unroll
  for (int r = 0; r < NG; ++r) {
    const int q = r * waves + w.wave;
    ne[r] = p.N - q * kE;
    bcq[r] = p.bc + (w.g * (long long)p.quads + (q < p.quads ? q : 0)) * p.ntok * 8;
#pragma unroll
    for (int e = 0; e < kE; ++e) A2[r][e] = h[r][e] = 0.f;
    states(p, w, q, [&](int e, long long at) { A2[r][e] = p.A[at] * kLog2e; });
    if (!STATE && p.chunks > 1)
      planes(p, w, q, [&](int e, long long at) { h[r][e] = p.ends[w.chunk * p.N * p.H + at]; });
  }
  const float bias = p.dbias != nullptr && w.in ? p.dbias[w.ch] : 0.f;
  const float skip = p.D != nullptr && w.in ? p.D[w.ch] : 0.f;
  float sumd = 0.f;
  bool dropped = false;
  Inputs<T> cur, next;
  auto hand_round = [&](const Inputs<T>& v, const Edges& ed, int buf) {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = w.wave + j * waves;
      if (i >= kL) continue;
      float dt = v.d[j] + bias;
      if (p.softplus) dt = softplus(dt);
      const bool ok = ed.valid >> i & 1;
      du[(buf * kL + i) * 64 + w.lane] = make_float2(ok ? dt : 0.f, ok ? dt * v.x[j] : 0.f);
      if (STATE) sumd += ok ? dt : 0.f;
    }
  };
  Edges ed = edges_of(p, w.c0, w.c1), ed_next = ed;
  cur.template load<false>(p, w, w.c0);
  hand_round(cur, ed, 0);
  __syncthreads();
  int buf = 0;
  for (int t = w.c0; t < w.c1; t += kL, buf ^= 1) {
    const bool more = t + kL < w.c1;
    if (more) {
      ed_next = edges_of(p, t + kL, w.c1);
      next.template load<false>(p, w, t + kL);
    }
    const float2* mine = du + buf * kL * 64 + w.lane;
    float* y_to = ys + ((buf * waves + w.wave) * kL) * 64 + w.lane;
    if (w.wave < active) {
      const bool edge = !ed.none();
      if (edge && (ed.start & 1)) {
        const long long s = (long long)seq_at(p, t) * p.H * p.N;
#pragma unroll
        for (int r = 0; r < NG; ++r) {
#pragma unroll
          for (int e = 0; e < kE; ++e) h[r][e] = 0.f;
          if (p.h0 != nullptr)
            states(p, w, r * waves + w.wave, [&](int e, long long at) { h[r][e] = p.h0[s + at]; });
        }
      }
      if (!STATE && p.saved != nullptr) {
        float* to = p.saved + (w.chunk * (p.len / kL) + (t - w.c0) / kL) * p.N * p.H;
#pragma unroll
        for (int r = 0; r < NG; ++r)
          planes(p, w, r * waves + w.wave, [&](int e, long long at) { to[at] = h[r][e]; });
      }
      auto token = [&](int i) {
        const float2 v = mine[i * 64];
        float y = 0.f;
#pragma unroll
        for (int r = 0; r < NG; ++r) {
          if (NG > 1 && r * waves + w.wave >= p.quads) continue;
          const F8 bc = bc_at(bcq[r] + (long long)(t + i) * 8);
          float a[kE];
          quad_step<PAD>(A2[r], bc, v.x, v.y, ne[r], h[r], a);
#pragma unroll
          for (int e = 0; e < kE; ++e) y = fmaf(bc[kE + e], h[r][e], y);
        }
        if (!STATE) y_to[i * 64] = y;
      };
      if (!edge) {
#pragma unroll
        for (int i = 0; i < kL; ++i) token(i);
      } else {
#pragma unroll 1
        for (int i = 0; i < kL && t + i < w.c1; ++i) {
          if ((ed.start >> i & 1) && i > 0) {
            const long long s = (long long)seq_at(p, t + i) * p.H * p.N;
#pragma unroll
            for (int r = 0; r < NG; ++r) {
#pragma unroll
              for (int e = 0; e < kE; ++e) h[r][e] = 0.f;
              if (p.h0 != nullptr)
                states(p, w, r * waves + w.wave, [&](int e, long long at) { h[r][e] = p.h0[s + at]; });
            }
          }
          token(i);
          if (!STATE && (ed.end >> i & 1)) {
            const long long s = (long long)seq_at(p, t + i) * p.H * p.N;
#pragma unroll
            for (int r = 0; r < NG; ++r)
              states(p, w, r * waves + w.wave, [&](int e, long long at) { p.hf[s + at] = h[r][e]; });
          }
        }
      }
    }
    dropped = dropped || ed.start != 0 || ed.valid != (1u << kL) - 1;
    if (more) hand_round(next, ed_next, buf ^ 1);
    __syncthreads();
    if (!STATE) {
      T* out = static_cast<T*>(p.out) + w.ch;
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int i = w.wave + j * waves;
        if (i >= kL || t + i >= w.c1 || !w.in) continue;
        float y = 0.f;
        for (int k = 0; k < active; ++k) y += ys[((buf * waves + k) * kL + i) * 64 + w.lane];
        y = fmaf(skip, cur.x[j], y);
        if (p.z != nullptr) y *= cur.z[j] * sigmoid(cur.z[j]);
        out[(long long)(t + i) * p.H] = (T)(ed.valid >> i & 1 ? y : 0.f);
      }
    }
    cur = next;
    ed = ed_next;
  }
  if (STATE) {
#pragma unroll
    for (int r = 0; r < NG; ++r)
      planes(p, w, r * waves + w.wave, [&](int e, long long at) { p.ends[w.chunk * p.N * p.H + at] = h[r][e]; });
    ys[w.wave * 64 + w.lane] = sumd;
    __syncthreads();
    if (w.wave == 0 && w.in) {
      float s = 0.f;
      for (int k = 0; k < waves; ++k) s += ys[k * 64 + w.lane];
      p.sumd[w.chunk * p.H + w.ch] = s;
    }
    if (w.g == 0 && w.hb == 0 && threadIdx.x == 0) p.drops[w.chunk] = dropped;
  }
}

// What enters each chunk, from what leaves the chunks before it, in their order (backward:
// after it, from the last).
template <bool BWD>
__global__ __launch_bounds__(256) void ssm_carry_kernel(SsmArgs p) {
  const long long hn = (long long)p.H * p.N;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.lines * hn) return;
  const long long line = i / hn, at = i - line * hn;
  const int n = (int)(at / p.H), ch = (int)(at - (long long)n * p.H);
  const float A2 = p.A[(long long)ch * p.N + n] * kLog2e;
  float carry = 0.f;
  for (int j = 0; j < p.chunks; ++j) {
    const long long c = line * p.chunks + (BWD ? p.chunks - 1 - j : j);
    const float e = p.ends[c * hn + at];
    p.ends[c * hn + at] = carry;
    carry = p.drops[c] ? e : fmaf(exp2_of(A2 * p.sumd[c * p.H + ch]), carry, e);
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// The sums over the 64 lanes of 64 values a lane, value l's in lane l. Each step halves the
// values: a lane keeps those whose bit is its own and adds what its partner has of them.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
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
template <class T, int NG, bool PAD>
__global__ __launch_bounds__(64 * kSsmWavesMax) void ssm_bwd_state_kernel(SsmArgs p) {
  extern __shared__ float shared[];
  float2* dd = reinterpret_cast<float2*>(shared);  // [2][kL][64]: step size, dy
  float* sums = shared + 2 * kL * 64 * 2;          // [waves][64]
  const Work w(p);
  const int waves = p.waves, active = p.quads < waves ? p.quads : waves;
  float A2[NG][kE], g[NG][kE];
  const float* bcq[NG];
  int ne[NG];
#pragma unroll
  for (int r = 0; r < NG; ++r) {
    const int q = r * waves + w.wave;
    ne[r] = p.N - q * kE;
    bcq[r] = p.bc + (w.g * (long long)p.quads + (q < p.quads ? q : 0)) * p.ntok * 8;
#pragma unroll
    for (int e = 0; e < kE; ++e) A2[r][e] = g[r][e] = 0.f;
    states(p, w, q, [&](int e, long long at) { A2[r][e] = p.A[at] * kLog2e; });
  }
  const float bias = p.dbias != nullptr && w.in ? p.dbias[w.ch] : 0.f;
  float sumd = 0.f;
  bool dropped = false;
  Inputs<T> cur;
  const int last = w.c0 + (w.c1 - 1 - w.c0) / kL * kL;
  int buf = 0;
  for (int t = last; t >= w.c0; t -= kL, buf ^= 1) {
    const Edges ed = edges_of(p, t, w.c1);
    cur.template load<true>(p, w, t);
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = w.wave + j * waves;
      if (i >= kL) continue;
      float dt = cur.d[j] + bias;
      if (p.softplus) dt = softplus(dt);
      float dy = cur.go[j];
      if (p.z != nullptr) dy *= cur.z[j] * sigmoid(cur.z[j]);
      const bool ok = ed.valid >> i & 1;
      dd[(buf * kL + i) * 64 + w.lane] = make_float2(ok ? dt : 0.f, ok ? dy : 0.f);
      sumd += ok ? dt : 0.f;
    }
    __syncthreads();
    const float2* mine = dd + buf * kL * 64 + w.lane;
    if (w.wave < active) {
      auto token = [&](int i) {
        const float2 v = mine[i * 64];
#pragma unroll
        for (int r = 0; r < NG; ++r) {
          if (NG > 1 && r * waves + w.wave >= p.quads) continue;
          const F8 bc = bc_at(bcq[r] + (long long)(t + i) * 8);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const bool no = PAD && e >= ne[r];
            g[r][e] = exp2_of((no ? 0.f : v.x) * A2[r][e]) * fmaf(bc[kE + e], no ? 0.f : v.y, g[r][e]);
          }
        }
      };
      if (ed.none()) {
#pragma unroll
        for (int i = kL - 1; i >= 0; --i) token(i);
      } else {
#pragma unroll 1
        for (int i = (w.c1 - t < kL ? w.c1 - t : kL) - 1; i >= 0; --i) {
          if (ed.end >> i & 1) {
            const long long s = (long long)seq_at(p, t + i) * p.H * p.N;
#pragma unroll
            for (int r = 0; r < NG; ++r) {
#pragma unroll
              for (int e = 0; e < kE; ++e) g[r][e] = 0.f;
              if (p.gh != nullptr)
                states(p, w, r * waves + w.wave, [&](int e, long long at) { g[r][e] = p.gh[s + at]; });
            }
          }
          token(i);
          if (ed.start >> i & 1) {
#pragma unroll
            for (int r = 0; r < NG; ++r)
#pragma unroll
              for (int e = 0; e < kE; ++e) g[r][e] = 0.f;
          }
        }
      }
    }
    dropped = dropped || ed.start != 0 || (t + kL <= w.c1 && ed.valid != (1u << kL) - 1);
  }
#pragma unroll
  for (int r = 0; r < NG; ++r)
    planes(p, w, r * waves + w.wave, [&](int e, long long at) { p.ends[w.chunk * p.N * p.H + at] = g[r][e]; });
  sums[w.wave * 64 + w.lane] = sumd;
  __syncthreads();
  if (w.wave == 0 && w.in) {
    float s = 0.f;
    for (int k = 0; k < waves; ++k) s += sums[k * 64 + w.lane];
    p.sumd[w.chunk * p.H + w.ch] = s;
  }
  if (w.g == 0 && w.hb == 0 && threadIdx.x == 0) p.drops[w.chunk] = dropped;
}

template <class T, int NG, bool PAD>
__global__ __launch_bounds__(64 * kSsmWavesMax) void ssm_bwd_kernel(SsmArgs p) {
  extern __shared__ float shared[];
  const int waves = p.waves, active = p.quads < waves ? p.quads : waves;
  float2* du = reinterpret_cast<float2*>(shared);            // [kL][64]: step size, times x
  float* dys = shared + kL * 64 * 2;                         // [kL][64]
  float2* s12 = reinterpret_cast<float2*>(dys + kL * 64);    // [waves][kL][64]
  float* s3 = dys + kL * 64 + waves * kL * 64 * 2;           // [waves][kL][64], with z only
  const Work w(p);
  const long long HN = (long long)p.H * p.N;
  float A2[NG][kE], g[NG][kE], dA[NG][kE];
#pragma unroll
  for (int r = 0; r < NG; ++r) {
    const int q = r * waves + w.wave;
#pragma unroll
    for (int e = 0; e < kE; ++e) A2[r][e] = g[r][e] = dA[r][e] = 0.f;
    states(p, w, q, [&](int e, long long at) { A2[r][e] = p.A[at] * kLog2e; });
    if (p.chunks > 1) planes(p, w, q, [&](int e, long long at) { g[r][e] = p.ends[w.chunk * HN + at]; });
  }
  const float bias = p.dbias != nullptr && w.in ? p.dbias[w.ch] : 0.f;
  const float skip = p.D != nullptr && w.in ? p.D[w.ch] : 0.f;
  float dD = 0.f, dbias = 0.f;
  const bool gated = p.z != nullptr;
  const int last = w.c0 + (w.c1 - 1 - w.c0) / kL * kL;
  for (int t = last; t >= w.c0; t -= kL) {
    const Edges ed = edges_of(p, t, w.c1);
    Inputs<T> in;
    in.template load<true>(p, w, t);
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = w.wave + j * waves;
      if (i >= kL) continue;
      float dt = in.d[j] + bias;
      if (p.softplus) dt = softplus(dt);
      float dy = in.go[j];
      if (gated) dy *= in.z[j] * sigmoid(in.z[j]);
      const bool ok = ed.valid >> i & 1;
      du[i * 64 + w.lane] = make_float2(ok ? dt : 0.f, ok ? dt * in.x[j] : 0.f);
      dys[i * 64 + w.lane] = ok ? dy : 0.f;
    }
    __syncthreads();
    if (w.wave < active) {
      const float* from = p.saved + (w.chunk * (p.len / kL) + (t - w.c0) / kL) * HN;
      auto quad = [&](auto edge_, auto round_) {
        constexpr bool EDGE = decltype(edge_)::value;
        constexpr int r = decltype(round_)::value;
        const int q = r * waves + w.wave;
        if (NG > 1 && q >= p.quads) return;
        const int ne = p.N - q * kE;
        const float* bcq = p.bc + ((w.g * (long long)p.quads + q) * p.ntok + t) * 8;
        float* to = p.part_bc == nullptr
                        ? nullptr
                        : p.part_bc +
                              (((w.hb * (long long)p.G + w.g) * p.quads + q) * p.ntok + t) * 8;
        // the batch's decays and the states before its tokens once more
        float a[kL][kE], hp[kL][kE], h[kE] = {};
        planes(p, w, q, [&](int e, long long at) { h[e] = from[at]; });
#pragma unroll
        for (int i = 0; i < kL; ++i) {
          if (EDGE && i > 0 && (ed.start >> i & 1)) {
            const long long s = (long long)seq_at(p, t + i) * HN;
#pragma unroll
            for (int e = 0; e < kE; ++e) h[e] = 0.f;
            if (p.h0 != nullptr) states(p, w, q, [&](int e, long long at) { h[e] = p.h0[s + at]; });
          }
#pragma unroll
          for (int e = 0; e < kE; ++e) hp[i][e] = h[e];
          const float2 v = du[i * 64 + w.lane];
          if (EDGE && !(ed.valid >> i & 1)) continue;
          quad_step<PAD>(A2[r], bc_at(bcq + i * 8), v.x, v.y, ne, h, a[i]);
        }
        float v64[64];
#pragma unroll
        for (int i = kL - 1; i >= 0; --i) {
          if (EDGE && (ed.end >> i & 1)) {
            const long long s = (long long)seq_at(p, t + i) * HN;
#pragma unroll
            for (int e = 0; e < kE; ++e) g[r][e] = 0.f;
            if (p.gh != nullptr) states(p, w, q, [&](int e, long long at) { g[r][e] = p.gh[s + at]; });
          }
          const int at = (w.wave * kL + i) * 64 + w.lane;
          const bool there = !EDGE || (ed.valid >> i & 1);
          float s1 = 0.f, s2 = 0.f, y = 0.f;
          if (!there) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v64[i % 8 * 8 + e] = 0.f;
          }
          if (there) {
          const float2 v = du[i * 64 + w.lane];
          const float dy = dys[i * 64 + w.lane];
          const F8 bc = bc_at(bcq + i * 8);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const bool no = PAD && e >= ne;
            // the state after the token: the next one's, unless a sequence begins there
            float ht;
            if (EDGE) ht = fmaf(a[i][e], hp[i][e], (no ? 0.f : v.y) * bc[e]);
            else ht = i + 1 < kL ? hp[i + 1 < kL ? i + 1 : 0][e] : h[e];
            const float d = fmaf(bc[kE + e], no ? 0.f : dy, g[r][e]);
            const float ga = a[i][e] * d;
            const float k = ga * hp[i][e];
            s1 = fmaf(bc[e], d, s1);
            s2 = fmaf(A2[r][e], k, s2);
            y = fmaf(bc[kE + e], ht, y);
            dA[r][e] = fmaf(no ? 0.f : v.x, k, dA[r][e]);
            v64[i % 8 * 8 + e] = d * v.y;
            v64[i % 8 * 8 + kE + e] = dy * ht;
            g[r][e] = ga;
          }
          }
          if (r == 0) {
            s12[at] = make_float2(s1, s2);
            if (gated) s3[at] = y;
          } else {
            s12[at] = make_float2(s12[at].x + s1, s12[at].y + s2);
            if (gated) s3[at] += y;
          }
          if (EDGE && (ed.start >> i & 1)) {
            const long long s = (long long)seq_at(p, t + i) * HN;
            if (p.gs != nullptr) states(p, w, q, [&](int e, long long at2) { p.gs[s + at2] = g[r][e]; });
#pragma unroll
            for (int e = 0; e < kE; ++e) g[r][e] = 0.f;
          }
          if (i % 8 == 0 && to != nullptr) {
            const float s = sum_lanes(v64, w.lane);
            if (!EDGE || t + i + w.lane / 8 < w.c1) to[i * 8 + w.lane] = s;
          }
        }
      };
      auto all = [&](auto edge_) {
        quad(edge_, std::integral_constant<int, 0>{});
        if constexpr (NG > 1) quad(edge_, std::integral_constant<int, 1>{});
      };
      if (ed.none()) all(std::false_type{});
      else all(std::true_type{});
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = w.wave + j * waves;
      if (i >= kL || t + i >= w.c1 || !w.in) continue;
      const long long at = (long long)(t + i) * p.H + w.ch;
      float s1 = 0.f, s2 = 0.f, y = 0.f;
      for (int k = 0; k < active; ++k) {
        const float2 q = s12[(k * kL + i) * 64 + w.lane];
        s1 += q.x;
        s2 += q.y;
        if (gated) y += s3[(k * kL + i) * 64 + w.lane];
      }
      const bool ok = ed.valid >> i & 1;
      const float x = in.x[j], dy = dys[i * 64 + w.lane], dt = du[i * 64 + w.lane].x;
      // s2 holds A in units of log2(e)
      float gd = fmaf(x, s1, s2 * (1.f / kLog2e));
      if (p.softplus) gd *= sigmoid(in.d[j] + bias);
      const float gx = fmaf(dt, s1, skip * dy);
      if (ok) {
        dD = fmaf(dy, x, dD);
        dbias += gd;
      }
      if (p.gx != nullptr) static_cast<T*>(p.gx)[at] = (T)(ok ? gx : 0.f);
      if (p.gd != nullptr) static_cast<T*>(p.gd)[at] = (T)(ok ? gd : 0.f);
      if (p.gz != nullptr) {
        const float z = in.z[j], sg = sigmoid(z);
        const float gz = in.go[j] * fmaf(skip, x, y) * sg * fmaf(z, 1.f - sg, 1.f);
        static_cast<T*>(p.gz)[at] = (T)(ok ? gz : 0.f);
      }
    }
    __syncthreads();
  }
  if (p.part_a != nullptr) {
#pragma unroll
    for (int r = 0; r < NG; ++r)
      planes(p, w, r * waves + w.wave, [&](int e, long long at) { p.part_a[w.chunk * HN + at] = dA[r][e]; });
  }
  if (p.part_h != nullptr) {
    shared[w.wave * 64 + w.lane] = dD;
    shared[(waves + w.wave) * 64 + w.lane] = dbias;
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
  const long long per = p.ntok * 8, total = (long long)p.G * p.quads * per;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float s = 0.f;
  for (int b = 0; b < p.hblocks; ++b) s += p.part_bc[b * total + i];
  const long long gq = i / per, rest = i - gq * per;
  const long long t = rest / 8;
  const int g = (int)(gq / p.quads), c = (int)(rest % 8);
  const int n = (int)(gq - (long long)g * p.quads) * kE + c % kE;
  if (n >= p.N) return;
  void* to = c < kE ? p.gB : p.gC;
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
  float s = 0.f;
  if (col < cols)
    for (long long i = part; i < items; i += kParts) s += from[i * stride];
  sums[part][threadIdx.x % kCols] = s;
  __syncthreads();
  if (part > 0 || col >= cols) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) s += sums[i][threadIdx.x];
  if (col < hn) {
    const long long n = col / p.H, c = col - n * p.H;
    if (p.gA != nullptr) p.gA[c * p.N + n] = s;
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

template <class T>
__global__ __launch_bounds__(kStepThreads) void ssm_step_kernel(SsmStepArgs p, int lanes) {
  const int row = blockIdx.y;
  const int lane = threadIdx.x & (lanes - 1);
  const int ch = blockIdx.x * (kStepThreads / lanes) + threadIdx.x / lanes;
  const bool in = ch < p.H;
  const int slot = p.slots != nullptr ? p.slots[row] : row;
  const bool live = slot >= 0 && slot < p.P;
  const int n0 = lane * kE, n = p.N - n0;
  const int g = in ? ch / (p.H / p.G) : 0;
  float* state = p.state + slot * p.ssp + (long long)ch * p.N + n0;
  Vec<float, kE> h{}, A{};
  float bias = 0.f, skip = 0.f;
  if (in && live) {
    if (n > 0) {
      h = load_vec<float, kE>(state, n);
      A = load_vec<float, kE>(p.A + (long long)ch * p.N + n0, n);
    }
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
  float f[kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) f[e] = h.get(e);
  auto step = [&](int r) {
    float y = 0.f, x = 0.f;
    if (in) {
      x = value(static_cast<const T*>(p.x) + r * p.sx + ch);
      float dt = value(static_cast<const T*>(p.d) + r * p.sd + ch) + bias;
      if (p.softplus) dt = softplus(dt);
      if (n > 0) {
        const Vec<T, kE> b = load_vec<T, kE>(static_cast<const T*>(p.Bm) + r * p.sbb + g * p.sbg + n0, n);
        const Vec<T, kE> c = load_vec<T, kE>(static_cast<const T*>(p.Cm) + r * p.scb + g * p.scg + n0, n);
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (e < n) {
            f[e] = fmaf(exp2_of(dt * (A.get(e) * kLog2e)), f[e], dt * x * b.get(e));
            y = fmaf(c.get(e), f[e], y);
          }
      }
    }
    for (int o = lanes / 2; o > 0; o /= 2) y += __shfl_xor(y, o);
    if (in && lane == 0) {
      y = fmaf(skip, x, y);
      if (p.z != nullptr) {
        const float z = value(static_cast<const T*>(p.z) + r * p.sz + ch);
        y *= z * sigmoid(z);
      }
      out[(long long)r * p.H] = (T)y;
    }
  };
  step(row);
  if (more)
    for (int r = row + 1; r < p.B; ++r)
      if (p.slots[r] == slot) step(r);
  if (in && n > 0) {
    h.put(f);
    store_vec<float, kE>(state, h, n);
  }
}

template <class F>
hipError_t with_type(int type, F&& f) {
  if (type == LTC_F32) return f(float{});
  if (type == LTC_BF16) return f(__bf16{});
  return f(_Float16{});
}

// Calls f with the rounds of quads and whether the last quad has states behind the last.
template <class F>
hipError_t with_states(const SsmArgs& a, F&& f) {
  using std::integral_constant;
  if (a.rounds == 1) {
    if (a.N % kE == 0) return f(integral_constant<int, 1>{}, std::false_type{});
    return f(integral_constant<int, 1>{}, std::true_type{});
  }
  if (a.N % kE == 0) return f(integral_constant<int, 2>{}, std::false_type{});
  return f(integral_constant<int, 2>{}, std::true_type{});
}

template <class T>
hipError_t launch_prep(const SsmArgs& a, const float* src, float* dst, hipStream_t s) {
  const long long n = a.ntok * a.G * a.quads, m = dst != nullptr ? (long long)a.B * a.H * a.N : 0;
  const long long blocks = ((n > m ? n : m) + 255) / 256;
  if (blocks == 0) return hipSuccess;
  LTC_LAUNCH((ssm_prep_kernel<T>), dim3((unsigned)(blocks > 16384 ? 16384 : blocks)), dim3(256), 0, s, a, src, dst);
  return hipGetLastError();
}

unsigned carry_groups(const SsmArgs& a) { return (unsigned)((a.lines * a.H * a.N + 255) / 256); }

}  // namespace

// Waves: four states each, at least four of them, at most eight, which take two quads each
// from 33 states on. A workgroup of four waves and 64 channels is one of a CU's two or
// three; with fewer than 512 in all, sequences are cut.
void ssm_plan(SsmArgs* a, bool packed) {
  a->quads = (a->N + kE - 1) / kE;
  a->rounds = a->quads > kSsmWavesMax ? 2 : 1;
  const int w = (a->quads + a->rounds - 1) / a->rounds;
  a->waves = w < kSsmWavesMin ? kSsmWavesMin : w;
  a->hblocks = (a->H / a->G + 63) / 64;
  a->lines = packed ? 1 : a->B;
  const long long base = a->lines * a->G * a->hblocks;
  long long chunks = 1;
  if (base > 0 && base < 256) chunks = (512 + base - 1) / base;
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
    hipError_t e = launch_prep<T>(a, a.h0, ends ? a.hf : nullptr, s);
    if (e != hipSuccess || a.ntok == 0) return e;
    return with_states(a, [&](auto ng, auto pad) {
      constexpr int NG = decltype(ng)::value;
      constexpr bool PAD = decltype(pad)::value;
      const dim3 grid((unsigned)(a.lines * a.chunks * a.G * a.hblocks)), block(64 * a.waves);
      const size_t lds = (2 * kL * 64 * 2 + 2 * a.waves * kL * 64) * sizeof(float);
      if (a.chunks > 1) {
        LTC_LAUNCH((ssm_fwd_kernel<T, NG, PAD, true>), grid, block, lds, s, a);
        LTC_LAUNCH((ssm_carry_kernel<false>), dim3(carry_groups(a)), dim3(256), 0, s, a);
      }
      LTC_LAUNCH((ssm_fwd_kernel<T, NG, PAD, false>), grid, block, lds, s, a);
      return hipGetLastError();
    });
  });
}

hipError_t launch_ssm_bwd(int type, const SsmArgs& a, hipStream_t s) {
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const bool ends = a.gs != nullptr && a.B > 0 && (a.cu != nullptr || a.ntok == 0);
    hipError_t e = launch_prep<T>(a, a.gh, ends ? a.gs : nullptr, s);
    if (e != hipSuccess) return e;
    if (a.ntok > 0) {
      e = with_states(a, [&](auto ng, auto pad) {
        constexpr int NG = decltype(ng)::value;
        constexpr bool PAD = decltype(pad)::value;
        const dim3 grid((unsigned)(a.lines * a.chunks * a.G * a.hblocks)), block(64 * a.waves);
        if (a.chunks > 1) {
          const size_t lds = (2 * kL * 64 * 2 + a.waves * 64) * sizeof(float);
          LTC_LAUNCH((ssm_bwd_state_kernel<T, NG, PAD>), grid, block, lds, s, a);
          LTC_LAUNCH((ssm_carry_kernel<true>), dim3(carry_groups(a)), dim3(256), 0, s, a);
        }
        const size_t lds = (kL * 64 * 3 + a.waves * kL * 64 * (a.z != nullptr ? 3 : 2)) * sizeof(float);
        LTC_LAUNCH((ssm_bwd_kernel<T, NG, PAD>), grid, block, lds, s, a);
        return hipGetLastError();
      });
      if (e != hipSuccess) return e;
      if (a.part_bc != nullptr) {
        const long long n = a.ntok * 8 * a.G * a.quads;
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
  while (lanes * kE < a.N) lanes *= 2;
  const int per = kStepThreads / lanes;
  const dim3 grid((a.H + per - 1) / per, a.B);
  return with_type(type, [&](auto t) {
    LTC_LAUNCH((ssm_step_kernel<decltype(t)>), grid, dim3(kStepThreads), 0, s, a, lanes);
    return hipGetLastError();
  });
}

}  // namespace ltc
