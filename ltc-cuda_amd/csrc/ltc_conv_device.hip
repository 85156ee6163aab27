// Short causal convolution of each channel, for gfx950:
//   pre_t = bias + sum_k w_k in_{t-K+1+k},   out_t = pre_t or silu(pre_t)
// where in is the sequence with its K-1 inputs before it (the state, or zeros).
// Backward, with d_t = dL/dout_t times silu'(pre_t) or 1:
//   dL/din_p = sum_j w_{K-1-j} d_{p+j},   dL/dw_k = sum_t d_t in_{t-K+1+k},   dL/dbias = sum_t d_t
//
// A thread walks a run of consecutive tokens with 16 bytes of channels and keeps the last
// K-1 inputs in registers, so each input is read once, but for the K-1 before a run. Bytes
// bound it. Taps are read once a run, in one stretch of memory per thread. The backward
// walks on K-1 tokens behind its run for the gradients that come from there, forms the
// slope again from the inputs, and leaves the sums of the weights' gradients tile by tile
// for a second launch, in the same order every time. Everything is summed in fp32 and
// rounded to its type once, when it is stored.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/ltc_capi.h"
#include "ltc_model_internal.h"
#include "ltc_tokens.h"
#include "ltc_vec.h"

namespace ltc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Tokens whose loads go out together.
constexpr int kAhead = 8;
// Bytes of a row per thread forward, channels per thread backward: the backward's sums
// and pending gradients, 3 K + 4 registers a channel, leave no room for eight.
constexpr int kFwdBytes = 16, kBwdChannels = 4;

__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -kLog2e));
}

// n values at p, of type T or fp32.
template <class T, int V>
__device__ __forceinline__ void load_weights(const void* base, long long at, int f32, int n, float (&d)[V]) {
  if (f32) {
    const Vec<float, V> q = load_vec<float, V>(static_cast<const float*>(base) + at, n);
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = q.get(i);
  } else {
    const Vec<T, V> q = load_vec<T, V>(static_cast<const T*>(base) + at, n);
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = q.get(i);
  }
}

// A thread's V channels: taps w[v * K + k], bias, and the inputs before the token at hand.
template <class T, int K, int V>
struct Channels {
  float w[V * K], bias[V];
  float win[K > 1 ? K - 1 : 1][V];

  __device__ __forceinline__ void taps(const void* wp, const void* bp, int f32, int ch, int n) {
    load_weights<T, V * K>(wp, (long long)ch * K, f32, n < V ? n * K : V * K, w);
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = 0.f;
    if (bp != nullptr) load_weights<T, V>(bp, ch, f32, n, bias);
  }
  // The inputs before token t of sequence q.
  __device__ __forceinline__ void before(const ConvArgs& p, const Seq& q, int t, int ch, int n) {
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      const int at = t - (K - 1) + i;
      Vec<T, V> r{};
      if (q.s >= 0) {
        if (at >= q.lo) r = load_vec<T, V>(static_cast<const T*>(p.x) + q.off + at * p.sxt + ch, n);
        else if (p.state != nullptr)
          r = load_vec<T, V>(static_cast<const T*>(p.state) +
                                 ((long long)q.s * (K - 1) + (K - 1 + at - q.lo)) * p.C + ch, n);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) win[i][v] = r.get(v);
    }
  }
  __device__ __forceinline__ float pre(const float (&x)[V], int v) const {
    float s = bias[v];
#pragma unroll
    for (int i = 0; i < K - 1; ++i) s = fmaf(w[v * K + i], win[i][v], s);
    return fmaf(w[v * K + K - 1], x[v], s);
  }
  __device__ __forceinline__ void push(const float (&x)[V]) {
#pragma unroll
    for (int i = 0; i + 1 < K - 1; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) win[i][v] = win[i + 1][v];
    if constexpr (K > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) win[K - 2][v] = x[v];
    }
  }
};

// Place of a workgroup and of a thread in it.
struct Place {
  long long tile;
  int cb, ch, n, slot;
  __device__ __forceinline__ Place(const ConvArgs& p, int V) {
    tile = blockIdx.x / (unsigned)p.cblocks;
    cb = (int)(blockIdx.x - tile * p.cblocks);
    ch = (cb * p.lanes + (int)(threadIdx.x & (p.lanes - 1))) * V;
    n = p.C - ch;
    slot = (int)threadIdx.x / p.lanes;
  }
};

template <class T, int K>
__global__ __launch_bounds__(kConvThreads) void conv_fwd_kernel(ConvArgs p) {
  constexpr int V = kFwdBytes / (int)sizeof(T);
  const Place at(p, V);
  const int ch = at.ch, n = at.n, slots = kConvThreads / p.lanes;
  if (n <= 0) return;
  const T* x = static_cast<const T*>(p.x) + ch;
  if (at.tile >= p.tiles) {
    // the last K-1 inputs of a sequence, its state's among them where it is short
    const int s = (int)(at.tile - p.tiles);
    int lo, hi;
    span_of(p.cu, p.T, (int)p.N, s, lo, hi);
    const long long off = p.cu == nullptr ? s * p.sxb - lo * p.sxt : 0;
    for (int i = at.slot; i < K - 1; i += slots) {
      const int t = hi - (K - 1) + i;
      Vec<T, V> r{};
      if (t >= lo) r = load_vec<T, V>(x + off + t * p.sxt, n);
      else if (p.state != nullptr)
        r = load_vec<T, V>(static_cast<const T*>(p.state) + ((long long)s * (K - 1) + (K - 1 + t - lo)) * p.C + ch,
                           n);
      store_vec<T, V>(static_cast<T*>(p.hf) + ((long long)s * (K - 1) + i) * p.C + ch, r, n);
    }
    return;
  }
  const long long first = (at.tile * slots + at.slot) * p.run;
  if (first >= p.N) return;
  int t = (int)first;
  const int end = (int)(first + p.run < p.N ? first + p.run : p.N);
  T* out = static_cast<T*>(p.out) + ch;
  Channels<T, K, V> c;
  c.taps(p.w, p.bias, p.w_f32, ch, n);
  Seq q = seq_of(p.cu, p.B, p.T, (int)p.N, t, p.sxb, p.sxt);
  c.before(p, q, t, ch, n);
  auto token = [&](const Vec<T, V>& xv, int u) {
    float f[V], o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = xv.get(v);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      o[v] = c.pre(f, v);
      if (p.silu) o[v] *= sigmoid(o[v]);
    }
    c.push(f);
    Vec<T, V> r;
    r.put(o);
    store_vec<T, V>(out + (long long)u * p.C, r, n);
  };
  while (t < end) {
    if (t >= q.hi) {
      q = seq_of(p.cu, p.B, p.T, (int)p.N, t, p.sxb, p.sxt);
      c.before(p, q, t, ch, n);
    }
    const T* px = x + q.off;
    if (q.s >= 0 && t + kAhead <= end && t + kAhead <= q.hi) {
      Vec<T, V> xv[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) xv[i] = load_vec<T, V>(px + (t + i) * p.sxt, n);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) token(xv[i], t + i);
      t += kAhead;
    } else if (q.s >= 0) {
      token(load_vec<T, V>(px + t * p.sxt, n), t);
      ++t;
    } else {
      store_vec<T, V>(out + (long long)t * p.C, Vec<T, V>{}, n);
      ++t;
    }
  }
}

// d_t of a token from its dL/dout.
template <class T, int K, int V>
__device__ __forceinline__ void slope_of(const Channels<T, K, V>& c, const float (&x)[V], int silu,
                                         float (&d)[V]) {
  if (!silu) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float y = c.pre(x, v), s = sigmoid(y);
    d[v] *= s * fmaf(y, 1.f - s, 1.f);
  }
}

template <class T, int K>
__global__ __launch_bounds__(kConvThreads) void conv_bwd_kernel(ConvArgs p) {
  constexpr int V = kBwdChannels;
  __shared__ float sums[kConvThreads * V];
  const Place at(p, V);
  const int ch = at.ch, n = at.n, slots = kConvThreads / p.lanes;
  const T* x = static_cast<const T*>(p.x) + ch;
  const T* go = static_cast<const T*>(p.go) + ch;
  Channels<T, K, V> c;
  if (at.tile >= p.tiles) {
    // the gradient of a sequence's state: of row i from the tokens up to the i-th, and
    // from the rows of the last inputs that are still the state's
    if (n <= 0 || at.slot > 0) return;
    c.taps(p.w, p.bias, p.w_f32, ch, n);
    const int s = (int)(at.tile - p.tiles);
    int lo, hi;
    span_of(p.cu, p.T, (int)p.N, s, lo, hi);
    Seq q{s, lo, hi, p.cu == nullptr ? s * p.sxb - lo * p.sxt : 0};
    const long long off = p.cu == nullptr ? s * p.sob - lo * p.sot : 0;
    c.before(p, q, lo, ch, n);
    float g[K > 1 ? K - 1 : 1][V];
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      Vec<T, V> r{};
      if (p.gh != nullptr && i >= hi - lo)
        r = load_vec<T, V>(static_cast<const T*>(p.gh) + ((long long)s * (K - 1) + i - (hi - lo)) * p.C + ch, n);
#pragma unroll
      for (int v = 0; v < V; ++v) g[i][v] = r.get(v);
    }
#pragma unroll
    for (int r = 0; r < K - 1; ++r) {
      if (p.go == nullptr || r >= hi - lo) continue;
      const Vec<T, V> xv = load_vec<T, V>(x + q.off + (lo + r) * p.sxt, n);
      const Vec<T, V> gv = load_vec<T, V>(go + off + (lo + r) * p.sot, n);
      float f[V], d[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[v] = xv.get(v);
        d[v] = gv.get(v);
      }
      slope_of(c, f, p.silu, d);
#pragma unroll
      for (int i = 0; i < K - 1; ++i)
        if (i >= r) {
#pragma unroll
          for (int v = 0; v < V; ++v) g[i][v] = fmaf(c.w[v * K + i - r], d[v], g[i][v]);
        }
      c.push(f);
    }
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      Vec<T, V> r;
      r.put(g[i]);
      store_vec<T, V>(static_cast<T*>(p.gs) + ((long long)s * (K - 1) + i) * p.C + ch, r, n);
    }
    return;
  }
  const long long first = (at.tile * slots + at.slot) * p.run;
  float dw[V * K], db[V];
#pragma unroll
  for (int i = 0; i < V * K; ++i) dw[i] = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) db[v] = 0.f;
  if (n > 0 && first < p.N) {
    const int t0 = (int)first, N = (int)p.N;
    const int end = (int)(first + p.run < p.N ? first + p.run : p.N);
    T* gx = static_cast<T*>(p.gx) + ch;
    c.taps(p.w, p.bias, p.w_f32, ch, n);
    int t = t0;
    Seq q = seq_of(p.cu, p.B, p.T, N, t, p.sxb, p.sxt);
    long long off = p.cu == nullptr ? q.s * p.sob - q.lo * p.sot : 0;
    c.before(p, q, t, ch, n);
    float pend[K][V];  // gradients of the inputs t - j, as far as they have come
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) pend[j][v] = 0.f;
    auto leave = [&](int u, const float (&g)[V]) {
      if (p.gx == nullptr || u < t0 || u >= end) return;
      Vec<T, V> r;
      r.put(g);
      store_vec<T, V>(gx + (long long)u * p.C, r, n);
    };
    // One token: its part of the weights' gradients where it is one of the run's (own),
    // and of the inputs' up to K-1 tokens before it, of its sequence (all: all of them).
    auto token = [&](const Vec<T, V>& xv, const Vec<T, V>& gv, int u, bool own, bool all) {
      float f[V], d[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f[v] = xv.get(v);
        d[v] = gv.get(v);
      }
      slope_of(c, f, p.silu, d);
      if (own) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          db[v] += d[v];
          dw[v * K + K - 1] = fmaf(d[v], f[v], dw[v * K + K - 1]);
#pragma unroll
          for (int k = 0; k < K - 1; ++k) dw[v * K + k] = fmaf(d[v], c.win[k][v], dw[v * K + k]);
        }
      }
      c.push(f);
#pragma unroll
      for (int j = K - 1; j > 0; --j)
#pragma unroll
        for (int v = 0; v < V; ++v) pend[j][v] = pend[j - 1][v];
#pragma unroll
      for (int v = 0; v < V; ++v) pend[0][v] = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (all || u - q.lo >= j) {
#pragma unroll
          for (int v = 0; v < V; ++v) pend[j][v] = fmaf(c.w[v * K + K - 1 - j], d[v], pend[j][v]);
        }
    };
    // the run, and the tokens behind it that its last inputs reach
    while (t < N && (t < end || (t < end + K - 1 && t < q.hi))) {
      if (t >= q.hi) {
        q = seq_of(p.cu, p.B, p.T, N, t, p.sxb, p.sxt);
        off = p.cu == nullptr ? q.s * p.sob - q.lo * p.sot : 0;
        c.before(p, q, t, ch, n);
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) pend[j][v] = 0.f;
      }
      if (q.s < 0) {
        const float none[V] = {};
        leave(t, none);
        ++t;
        continue;
      }
      const T* px = x + q.off;
      const T* pg = go + off;
      if (p.go != nullptr && t + kAhead <= end && t + kAhead < q.hi && t - q.lo >= K - 1) {
        Vec<T, V> xv[kAhead], gv[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          xv[i] = load_vec<T, V>(px + (t + i) * p.sxt, n);
          gv[i] = load_vec<T, V>(pg + (t + i) * p.sot, n);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          token(xv[i], gv[i], t + i, true, true);
          leave(t + i - (K - 1), pend[K - 1]);
        }
        t += kAhead;
        continue;
      }
      const Vec<T, V> xv = load_vec<T, V>(px + t * p.sxt, n);
      Vec<T, V> gv{};
      if (p.go != nullptr) gv = load_vec<T, V>(pg + t * p.sot, n);
      token(xv, gv, t, t < end, false);
      if (t - (K - 1) >= q.lo) leave(t - (K - 1), pend[K - 1]);
      ++t;
      if (t == q.hi) {
        // the sequence's last inputs, which are also its final state
#pragma unroll
        for (int j = K - 2; j >= 0; --j) {
          const int u = t - 1 - j;
          if (u < q.lo) continue;
          if (p.gh != nullptr) {
            const Vec<T, V> r = load_vec<T, V>(
                static_cast<const T*>(p.gh) + ((long long)q.s * (K - 1) + (K - 2 - j)) * p.C + ch, n);
#pragma unroll
            for (int v = 0; v < V; ++v) pend[j][v] += r.get(v);
          }
          leave(u, pend[j]);
        }
      }
    }
  }
  if (p.part == nullptr) return;
  // the slots' sums, slot by slot
  const int width = p.lanes * V;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v)
      sums[at.slot * width + (int)(threadIdx.x & (p.lanes - 1)) * V + v] = k < K ? dw[v * K + (k < K ? k : 0)] : db[v];
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += kConvThreads) {
      const int cc = at.cb * width + i;
      float s = 0.f;
      for (int j = 0; j < slots; ++j) s += sums[j * width + i];
      if (cc < p.C) p.part[(at.tile * (K + 1) + k) * p.C + cc] = s;
    }
  }
}

// The tiles' sums, in kParts interleaved parts.
template <class T>
__global__ __launch_bounds__(kConvThreads) void conv_sum_kernel(ConvArgs p, int K) {
  constexpr int kCols = 32, kParts = kConvThreads / kCols;
  __shared__ float sums[kParts][kCols];
  const long long cols = (long long)(K + 1) * p.C;
  const long long col = (long long)blockIdx.x * kCols + threadIdx.x % kCols;
  const int part = threadIdx.x / kCols;
  float s = 0.f;
  if (col < cols)
    for (long long i = part; i < p.tiles; i += kParts) s += p.part[i * cols + col];
  sums[part][threadIdx.x % kCols] = s;
  __syncthreads();
  if (part > 0 || col >= cols) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kParts; ++i) s += sums[i][threadIdx.x];
  const int k = (int)(col / p.C);
  const long long c = col - (long long)k * p.C;
  void* to = k < K ? p.gw : p.gb;
  if (to == nullptr) return;
  const long long at = k < K ? c * K + k : c;
  if (p.w_f32) static_cast<float*>(to)[at] = s;
  else static_cast<T*>(to)[at] = (T)s;
}

constexpr int kStepThreads = 64;
constexpr int kStepChannels = 4;

template <class T, int K>
__global__ __launch_bounds__(kStepThreads) void conv_step_kernel(ConvStepArgs p) {
  constexpr int V = kStepChannels;
  const int row = blockIdx.y;
  const int ch = (blockIdx.x * kStepThreads + threadIdx.x) * V;
  const int n = p.C - ch;
  const int slot = p.slots != nullptr ? p.slots[row] : row;
  const bool live = slot >= 0 && slot < p.P;
  T* out = static_cast<T*>(p.out) + ch;
  T* state = static_cast<T*>(p.state) + slot * p.ssp + ch;
  const T* x = static_cast<const T*>(p.x) + ch;
  Channels<T, K, V> c;
  Vec<T, V> xv{}, win[K > 1 ? K - 1 : 1];
  if (n > 0 && live) {
    xv = load_vec<T, V>(x + row * p.sxb, n);
#pragma unroll
    for (int i = 0; i < K - 1; ++i) win[i] = load_vec<T, V>(state + i * p.sst, n);
    c.taps(p.w, p.bias, p.w_f32, ch, n);
  }
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
      if (n > 0) store_vec<T, V>(out + (long long)row * p.C, o, n);
      return;
    }
    if (earlier) return;
  }
  if (n <= 0) return;
#pragma unroll
  for (int i = 0; i < K - 1; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) c.win[i][v] = win[i].get(v);
  auto step = [&](int r) {
    float f[V], o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = xv.get(v);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      o[v] = c.pre(f, v);
      if (p.silu) o[v] *= sigmoid(o[v]);
    }
    c.push(f);
    Vec<T, V> q;
    q.put(o);
    store_vec<T, V>(out + (long long)r * p.C, q, n);
  };
  step(row);
  if (more)
    for (int r = row + 1; r < p.B; ++r) {
      if (p.slots[r] != slot) continue;
      xv = load_vec<T, V>(x + r * p.sxb, n);
      step(r);
    }
#pragma unroll
  for (int i = 0; i < K - 1; ++i) {
    Vec<T, V> q;
    q.put(c.win[i]);
    store_vec<T, V>(state + i * p.sst, q, n);
  }
}

template <class F>
hipError_t with_type(int x_type, F&& f) {
  if (x_type == LTC_F32) return f(float{});
  if (x_type == LTC_BF16) return f(__bf16{});
  return f(_Float16{});
}

// Calls f with K as a constant.
template <class F>
hipError_t with_taps(int K, F&& f) {
  switch (K) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}

}  // namespace

// Runs of 8 to 64 tokens: as long as 4096 waves are left of them, since every run reads
// K-1 tokens more at each end.
void conv_tiles(int x_type, bool bwd, ConvArgs* a) {
  const int V = bwd ? kBwdChannels : kFwdBytes / (x_type == LTC_F32 ? 4 : 2);
  const long long vecs = (a->C + V - 1) / V;
  int lanes = 8;
  while (lanes < 64 && lanes < vecs) lanes *= 2;
  a->lanes = lanes;
  a->cblocks = (int)((vecs + lanes - 1) / lanes);
  const long long waves = (vecs * a->N + 63) / 64 / kAhead;
  const long long r = waves / 4096;
  a->run = kAhead * (int)(r < 1 ? 1 : r > 8 ? 8 : r);
  const long long per = (long long)(kConvThreads / lanes) * a->run;
  a->tiles = (a->N + per - 1) / per;
}

hipError_t launch_conv_fwd(int x_type, int K, const ConvArgs& a, hipStream_t s) {
  const long long groups = (a.tiles + (K > 1 ? a.B : 0)) * a.cblocks;
  if (groups == 0) return hipSuccess;
  return with_type(x_type, [&](auto t) {
    using T = decltype(t);
    return with_taps(K, [&](auto k) {
      LTC_LAUNCH((conv_fwd_kernel<T, decltype(k)::value>), dim3((unsigned)groups), dim3(kConvThreads), 0, s, a);
      return hipGetLastError();
    });
  });
}

hipError_t launch_conv_bwd(int x_type, int K, const ConvArgs& a, hipStream_t s) {
  return with_type(x_type, [&](auto t) {
    using T = decltype(t);
    const long long groups = (a.tiles + (K > 1 && a.gs != nullptr ? a.B : 0)) * a.cblocks;
    hipError_t e = hipSuccess;
    if (groups > 0)
      e = with_taps(K, [&](auto k) {
        LTC_LAUNCH((conv_bwd_kernel<T, decltype(k)::value>), dim3((unsigned)groups), dim3(kConvThreads), 0, s, a);
        return hipGetLastError();
      });
    if (e != hipSuccess || (a.gw == nullptr && a.gb == nullptr)) return e;
    const unsigned sums = (unsigned)(((long long)(K + 1) * a.C + 31) / 32);
    LTC_LAUNCH((conv_sum_kernel<T>), dim3(sums), dim3(kConvThreads), 0, s, a, K);
    return hipGetLastError();
  });
}

hipError_t launch_conv_step(int x_type, int K, const ConvStepArgs& a, hipStream_t s) {
  if (a.B == 0) return hipSuccess;
  constexpr int per = kStepThreads * kStepChannels;
  const dim3 grid((a.C + per - 1) / per, a.B);
  return with_type(x_type, [&](auto t) {
    using T = decltype(t);
    return with_taps(K, [&](auto k) {
      LTC_LAUNCH((conv_step_kernel<T, decltype(k)::value>), grid, dim3(kStepThreads), 0, s, a);
      return hipGetLastError();
    });
  });
}

}  // namespace ltc
