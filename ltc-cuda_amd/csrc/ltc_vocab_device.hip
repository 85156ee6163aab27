// What joins a model to its vocabulary, for gfx950: the embedding's rows with the gradient
// of its table, and the adjustments of logits before a token is chosen.
//
// Embedding: out_i = scale table[ids_i]. Its gradient, of row v: scale times the sum of
// dL/dout_i over the i with ids_i = v. The ids are sorted by a stable radix sort that
// carries their places, so that each row's gradient is one run of places in ascending
// order, summed in fp32 and rounded once: the same bits every time, each row of dL/dout
// read once and each row of the gradient written once. A run that is long (a frequent id)
// is cut at multiples of kEmbedPiece sorted ids: pieces inside one run are summed by
// workgroups of their own, and the row adds their sums in order.
//
// Adjustments: one pass over the logits. A workgroup has a segment of a row, counts the
// context's ids of its segment in shared memory, and leaves the few biased logits, which
// it knows from a list, for the end. Bytes bound both.
#include <hip/hip_runtime.h>

#include "../../include/ltc_capi.h"
#include "ltc_model_internal.h"
#include "ltc_vec.h"

namespace ltc {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ long long id_at(const void* ids, int id64, long long i) {
  return id64 ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------
// `lanes` threads to a row.
template <class T>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(EmbedArgs p, int lanes) {
  constexpr int V = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & (lanes - 1);
  const long long row = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  if (row >= p.n) return;
  const long long id = id_at(p.ids, p.id64, row);
  const T* from = static_cast<const T*>(p.table) + id * p.st;
  T* to = static_cast<T*>(p.out) + row * p.H;
  const bool there = id >= 0 && id < p.V;
  for (int c = lane * V; c < p.H; c += lanes * V) {
    const int n = p.H - c;
    float f[V];
    if (there) {
      const Vec<T, V> r = load_vec<T, V>(from + c, n);
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = r.get(v) * p.scale;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = id < 0 ? 0.f : __builtin_nanf("");
    }
    Vec<T, V> o;
    o.put(f);
    store_vec<T, V>(to + c, o, n);
  }
}

// An id as it is sorted: those that are not in the table come last.
__device__ __forceinline__ int key_of(const EmbedArgs& p, long long i) {
  const long long id = id_at(p.ids, p.id64, i);
  return id >= 0 && id < p.V ? (int)id : p.V;
}

__device__ __forceinline__ void forget_runs(const EmbedArgs& p) {
  for (long long v = (long long)blockIdx.x * kSortThreads + threadIdx.x; v < p.V;
       v += (long long)gridDim.x * kSortThreads)
    p.begin[v] = -1;
}

// Counts of a tile's digits. The first pass also forgets the runs of an earlier call.
__global__ __launch_bounds__(kSortThreads) void embed_count_kernel(EmbedArgs p, int pass) {
  __shared__ unsigned hist[1 << kSortBitsMax];
  const int buckets = 1 << p.bits, shift = pass * p.bits;
  if (pass == 0) forget_runs(p);
  for (int d = threadIdx.x; d < buckets; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * kSortTile;
#pragma unroll
  for (int i = 0; i < kSortTile / kSortThreads; ++i) {
    const long long at = first + i * kSortThreads + threadIdx.x;
    if (at < p.n) {
      const int k = pass == 0 ? key_of(p, at) : p.key[(pass - 1) & 1][at];
      atomicAdd(&hist[k >> shift & (buckets - 1)], 1u);
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < buckets; d += kSortThreads)
    p.counts[(long long)blockIdx.x * buckets + d] = hist[d];
}

// Of many tiles: each count is replaced by the digit's counts in the tiles before, and
// the digit's total is left behind the last tile's.
__global__ __launch_bounds__(64) void embed_scan_kernel(EmbedArgs p) {
  const int buckets = 1 << p.bits, d = blockIdx.x * 64 + threadIdx.x;
  if (d >= buckets) return;
  constexpr int kAhead = 32;  // under way together
  unsigned sum = 0;
  for (int t0 = 0; t0 < p.tiles; t0 += kAhead) {
    unsigned c[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) c[j] = p.counts[(long long)min(t0 + j, p.tiles - 1) * buckets + d];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (t0 + j >= p.tiles) break;
      p.counts[(long long)(t0 + j) * buckets + d] = sum;
      sum += c[j];
    }
  }
  p.counts[(long long)p.tiles * buckets + d] = sum;
}

struct SortShared {
  static constexpr int kWaves = kSortThreads / 64;
  unsigned short hist[kWaves][1 << kSortBitsMax];  // at most the tile's ids
  unsigned base[1 << kSortBitsMax];
  unsigned sums[kWaves];
};

// One pass over one tile. The place of an id among those of its digit: those of the tiles
// before, of the waves before, and of the ids before in its wave, which owns consecutive
// ids and takes them 64 at a time.
__device__ __forceinline__ void sort_tile(const EmbedArgs& p, SortShared& sh, int tile, int pass, bool direct) {
  constexpr int kRounds = kSortTile / kSortThreads;
  const int buckets = 1 << p.bits, shift = pass * p.bits;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int d = threadIdx.x;  // a thread's own digit
  for (int i = lane; i < buckets; i += 64) sh.hist[wave][i] = 0;
  int key[kRounds], pos[kRounds], rank[kRounds];
  const long long first = (long long)tile * kSortTile + wave * (64 * kRounds) + lane;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const long long at = first + i * 64;
    const bool in = at < p.n;
    key[i] = 0;
    pos[i] = 0;
    if (in) {
      key[i] = pass == 0 ? key_of(p, at) : p.key[(pass - 1) & 1][at];
      pos[i] = pass == 0 ? (int)at : p.pos[(pass - 1) & 1][at];
    }
    const int digit = key[i] >> shift & (buckets - 1);
    unsigned long long same = __ballot(in);
    for (int b = 0; b < p.bits; ++b) {
      const unsigned long long bal = __ballot(digit >> b & 1);
      same &= digit >> b & 1 ? bal : ~bal;
    }
    const int before = __popcll(same & ((1ull << lane) - 1));
    unsigned old = 0;
    if (in) old = sh.hist[wave][digit];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && before == 0) sh.hist[wave][digit] = (unsigned short)(old + __popcll(same));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    rank[i] = (int)old + before;
  }
  __syncthreads();
  // counts of the digit: in the tiles before (lower), in all (total), in the waves before
  unsigned lower = 0, total = 0;
  if (d < buckets) {
    if (p.tiles == 1) {
#pragma unroll
      for (int w = 0; w < SortShared::kWaves; ++w) total += sh.hist[w][d];
    } else if (direct) {
      constexpr int kAhead = 16;
      for (int t0 = 0; t0 < p.tiles; t0 += kAhead) {
        unsigned c[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) c[j] = p.counts[(long long)min(t0 + j, p.tiles - 1) * buckets + d];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (t0 + j < tile) lower += c[j];
          if (t0 + j < p.tiles) total += c[j];
        }
      }
    } else {
      lower = p.counts[(long long)tile * buckets + d];
      total = p.counts[(long long)p.tiles * buckets + d];
    }
    unsigned run = 0;
#pragma unroll
    for (int w = 0; w < SortShared::kWaves; ++w) {
      const unsigned c = sh.hist[w][d];
      sh.hist[w][d] = (unsigned short)run;
      run += c;
    }
  }
  // totals of the digits below, by waves and then across them
  unsigned up = total;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const unsigned q = __shfl_up(up, o);
    if (lane >= o) up += q;
  }
  if (lane == 63) sh.sums[wave] = up;
  __syncthreads();
  unsigned below = up - total;
  for (int w = 0; w < wave; ++w) below += sh.sums[w];
  if (d < buckets) sh.base[d] = below + lower;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (first + i * 64 >= p.n) continue;
    const int digit = key[i] >> shift & (buckets - 1);
    const unsigned to = sh.base[digit] + sh.hist[wave][digit] + (unsigned)rank[i];
    p.key[pass & 1][to] = key[i];
    p.pos[pass & 1][to] = pos[i];
  }
}

__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedArgs p, int pass, bool direct) {
  __shared__ SortShared sh;
  sort_tile(p, sh, blockIdx.x, pass, direct);
}

// All passes over ids that one workgroup holds.
__global__ __launch_bounds__(kSortThreads) void embed_sort_one_kernel(EmbedArgs p) {
  __shared__ SortShared sh;
  forget_runs(p);
  for (int pass = 0; pass < p.passes; ++pass) {
    sort_tile(p, sh, 0, pass, true);
    __syncthreads();
  }
}

// Rows of dL/dout at the sorted places lo up to hi, added to f in their order.
template <class T, int V>
__device__ __forceinline__ void add_rows(const EmbedArgs& p, const int* pos, int lo, int hi, int c, int n,
                                         float (&f)[V]) {
  constexpr int kRows = 8;  // under way together
  const T* go = static_cast<const T*>(p.go) + c;
  int i = lo;
  for (; i + kRows <= hi; i += kRows) {
    Vec<T, V> r[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) r[j] = load_vec<T, V>(go + pos[i + j] * p.sgo, n);
#pragma unroll
    for (int j = 0; j < kRows; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] += r[j].get(v);
  }
  for (; i < hi; ++i) {
    const Vec<T, V> r = load_vec<T, V>(go + pos[i] * p.sgo, n);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] += r.get(v);
  }
}

// A piece of the sorted ids: where runs begin and end in it, and its sum where it is all
// of one run.
template <class T>
__global__ __launch_bounds__(kThreads) void embed_piece_kernel(EmbedArgs p, int cblocks) {
  constexpr int V = 16 / (int)sizeof(T);
  const int piece = blockIdx.x / (unsigned)cblocks, cb = blockIdx.x % (unsigned)cblocks;
  const int* key = p.key[(p.passes - 1) & 1];
  const int* pos = p.pos[(p.passes - 1) & 1];
  const int lo = piece * kEmbedPiece;
  const int hi = (int)(p.n - lo < kEmbedPiece ? p.n : lo + kEmbedPiece);
  if (cb == 0 && (int)threadIdx.x < hi - lo) {
    const int i = lo + threadIdx.x, k = key[i];
    if (k < p.V) {
      if (i == 0 || key[i - 1] != k) p.begin[k] = i;
      if (i + 1 == p.n || key[i + 1] != k) p.end[k] = i + 1;
    }
  }
  if (hi - lo < kEmbedPiece || key[lo] != key[hi - 1] || key[lo] >= p.V) return;
  const int c = (cb * kThreads + (int)threadIdx.x) * V, n = p.H - c;
  if (n <= 0) return;
  float f[V] = {};
  add_rows<T, V>(p, pos, lo, hi, c, n, f);
  Vec<float, V> o;
  o.put(f);
  store_vec<float, V>(p.sums + (long long)piece * p.H + c, o, n);
}

// Rows of the gradient, `lanes` threads to each. A row is a chain of loads, of its run's
// ends, its places and its rows, so what counts is how many rows are at work at once: few
// registers, and one row to a thread (four, their ends read together, took 162 us for
// 92 at 65536 rows of 2048 bf16; a wave to a row 203).
template <class T>
__global__ __launch_bounds__(kThreads, 8) void embed_rows_kernel(EmbedArgs p, int lanes) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int kSums = 4;  // of pieces, under way together
  const int lane = threadIdx.x & (lanes - 1);
  const long long row = (long long)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  if (row >= p.V) return;
  const int* pos = p.pos[(p.passes - 1) & 1];
  int lo = -1, hi = -1;
  if (p.n > 0) {
    lo = p.begin[row];
    hi = p.end[row];  // of an id that does not occur, anything
  }
  // whole pieces between, if any
  const int p0 = (lo + kEmbedPiece - 1) / kEmbedPiece, p1 = hi / kEmbedPiece;
  T* to = static_cast<T*>(p.gt) + row * p.H;
  for (int c = lane * V; c < p.H; c += lanes * V) {
    const int n = p.H - c;
    float f[V] = {};
    if (lo >= 0) {
      if (p0 >= p1) {
        add_rows<T, V>(p, pos, lo, hi, c, n, f);
      } else {
        add_rows<T, V>(p, pos, lo, p0 * kEmbedPiece, c, n, f);
        const float* sums = p.sums + c;
        for (int i = p0; i < p1; i += kSums) {
          Vec<float, V> s[kSums];
#pragma unroll
          for (int k = 0; k < kSums; ++k)
            s[k] = load_vec<float, V>(sums + (long long)min(i + k, p1 - 1) * p.H, n);
#pragma unroll
          for (int k = 0; k < kSums; ++k)
            if (i + k < p1) {
#pragma unroll
              for (int v = 0; v < V; ++v) f[v] += s[k].get(v);
            }
        }
        add_rows<T, V>(p, pos, p1 * kEmbedPiece, hi, c, n, f);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] *= p.scale;
    }
    Vec<T, V> o;
    o.put(f);
    store_vec<T, V>(to + c, o, n);
  }
}

int row_lanes(int H, int V, int most) {
  int lanes = 1;
  while (lanes < most && lanes * V < H) lanes *= 2;
  return lanes;
}

template <class F>
hipError_t with_type(int type, F&& f) {
  if (type == LTC_F32) return f(float{});
  if (type == LTC_BF16) return f(__bf16{});
  return f(_Float16{});
}

// ---------------------------------------------------------------------------
// Adjustments of logits
// ---------------------------------------------------------------------------
// Count of an id: whether it occurs at all, and how often behind the prompt.
constexpr unsigned kSeen = 0x80000000u;

__device__ __forceinline__ float adjusted(float x, unsigned c, float rep, float freq, float pres) {
  if (c == 0) return x;
  x = x > 0.f ? x / rep : x * rep;
  const unsigned often = c & ~kSeen;
  if (often > 0) {
    x -= freq * (float)often;
    x -= pres;
  }
  return x;
}

__device__ __forceinline__ bool allowed(const int* mask, int v) { return mask[v >> 5] >> (v & 31) & 1; }

template <class T>
__global__ __launch_bounds__(kThreads) void adjust_kernel(AdjustArgs p) {
  constexpr int V = 16 / (int)sizeof(T);
  extern __shared__ __attribute__((aligned(16))) unsigned count[];
  const long long row = blockIdx.x / (unsigned)p.segs;
  const int lo = (int)(blockIdx.x % (unsigned)p.segs) * p.seg;
  const int len = p.V - lo < p.seg ? p.V - lo : p.seg;
  const float rep = p.rep != nullptr ? p.rep[row] : p.rep0;
  const float freq = p.freq != nullptr ? p.freq[row] : p.freq0;
  const float pres = p.pres != nullptr ? p.pres[row] : p.pres0;
  const T* x = static_cast<const T*>(p.logits) + row * p.sl + lo;
  T* out = static_cast<T*>(p.out) + row * p.V + lo;
  const int* mask = p.mask != nullptr ? p.mask + row * p.sm + lo / 32 : nullptr;
  // The first logits are under way while the context is counted.
  constexpr int kAhead = 4;
  Vec<T, V> r[kAhead];
  const auto get = [&](int i) { return i < len ? load_vec<T, V>(x + i, len - i) : Vec<T, V>{}; };
#pragma unroll
  for (int j = 0; j < kAhead; ++j) r[j] = get((j * kThreads + (int)threadIdx.x) * V);
  if (p.ctx > 0) {
    for (int i = threadIdx.x; i < p.seg; i += kThreads) count[i] = 0;
    __syncthreads();
    const int prompt = p.prompt != nullptr ? p.prompt[row] : 0;
    constexpr int kIds = 8;  // of a thread, under way together
    for (int i0 = threadIdx.x; i0 < p.ctx; i0 += kIds * kThreads) {
      long long id[kIds];
#pragma unroll
      for (int j = 0; j < kIds; ++j)
        id[j] = id_at(p.context, p.ctx64, row * p.sc + min(i0 + j * kThreads, p.ctx - 1));
#pragma unroll
      for (int j = 0; j < kIds; ++j) {
        const int i = i0 + j * kThreads;
        if (i >= p.ctx || id[j] < lo || id[j] >= (long long)lo + len) continue;
        atomicOr(&count[id[j] - lo], kSeen);
        if (i >= prompt) atomicAdd(&count[id[j] - lo], 1u);
      }
    }
    __syncthreads();
  }
  for (int i0 = threadIdx.x * V; i0 < len; i0 += kAhead * kThreads * V) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kThreads * V;
      if (i >= len) continue;
      const unsigned bits = mask != nullptr ? (unsigned)mask[i >> 5] >> (i & 31) : ~0u;
      float f[V];
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = r[j].get(v);
      if (p.ctx > 0) {
        unsigned c[V], any = 0;
        __builtin_memcpy(c, __builtin_assume_aligned(count + i, 16), sizeof(c));
#pragma unroll
        for (int v = 0; v < V; ++v) any |= c[v];
        if (any != 0) {
#pragma unroll
          for (int v = 0; v < V; ++v) f[v] = adjusted(f[v], c[v], rep, freq, pres);
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (!(bits >> v & 1)) f[v] = -__builtin_inff();
      Vec<T, V> o;
      o.put(f);
      store_vec<T, V>(out + i, o, len - i);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) r[j] = get(i0 + (kAhead + j) * kThreads * V);
  }
  if (p.K == 0) return;
  // The biased logits once more: an id's first entry takes all of its entries, in order.
  // An entry looks for its id in those before it, load by load: fine for some tens of
  // biases; for hundreds it outlasts the rest of a small call.
  __syncthreads();
  for (int k = threadIdx.x; k < p.K; k += kThreads) {
    const long long id = id_at(p.bias_ids, p.bias64, row * p.sbi + k);
    if (id < lo || id >= (long long)lo + len) continue;
    bool first = true;
    for (int j = 0; j < k && first; ++j) first = id_at(p.bias_ids, p.bias64, row * p.sbi + j) != id;
    if (!first) continue;
    float b = p.bias[row * p.sb + k];
    for (int j = k + 1; j < p.K; ++j)
      if (id_at(p.bias_ids, p.bias64, row * p.sbi + j) == id) b += p.bias[row * p.sb + j];
    const int v = (int)(id - lo);
    float f = (float)x[v];
    if (p.ctx > 0) f = adjusted(f, count[v], rep, freq, pres);
    f += b;
    if (mask != nullptr && !allowed(mask, v)) f = -__builtin_inff();
    out[v] = (T)f;
  }
}

}  // namespace

void embed_digits(EmbedArgs* a) {
  int bits = 1;
  while (bits < 32 && (1ll << bits) <= a->V) ++bits;
  a->passes = (bits + kSortBitsMax - 1) / kSortBitsMax;
  a->bits = (bits + a->passes - 1) / a->passes;
}

hipError_t launch_embed_fwd(int type, const EmbedArgs& a, hipStream_t s) {
  if (a.n == 0) return hipSuccess;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    const int lanes = row_lanes(a.H, 16 / (int)sizeof(T), kThreads), rows = kThreads / lanes;
    LTC_LAUNCH((embed_fwd_kernel<T>), dim3((unsigned)((a.n + rows - 1) / rows)), dim3(kThreads), 0, s, a, lanes);
    return hipGetLastError();
  });
}

hipError_t launch_embed_bwd(int type, const EmbedArgs& a, hipStream_t s) {
  if (a.n > 0 && a.tiles == 1) {
    LTC_LAUNCH(embed_sort_one_kernel, dim3(1), dim3(kSortThreads), 0, s, a);
  } else if (a.n > 0) {
    const bool direct = a.tiles <= kSortTilesDirect;
    const dim3 grid((unsigned)a.tiles), block(kSortThreads);
    for (int pass = 0; pass < a.passes; ++pass) {
      LTC_LAUNCH(embed_count_kernel, grid, block, 0, s, a, pass);
      if (!direct) LTC_LAUNCH(embed_scan_kernel, dim3(((1u << a.bits) + 63) / 64), dim3(64), 0, s, a);
      LTC_LAUNCH(embed_sort_kernel, grid, block, 0, s, a, pass, direct);
    }
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / (int)sizeof(T);
    if (a.n > 0) {
      const int cblocks = (int)(((long long)a.H + kThreads * V - 1) / (kThreads * V));
      const long long pieces = (a.n + kEmbedPiece - 1) / kEmbedPiece;
      LTC_LAUNCH((embed_piece_kernel<T>), dim3((unsigned)(pieces * cblocks)), dim3(kThreads), 0, s, a, cblocks);
    }
    const int lanes = row_lanes(a.H, V, kThreads), rows = kThreads / lanes;
    LTC_LAUNCH((embed_rows_kernel<T>), dim3((unsigned)(((long long)a.V + rows - 1) / rows)), dim3(kThreads), 0, s, a,
               lanes);
    return hipGetLastError();
  });
}

// Segments of 1024 to 8192 logits, as long as 2048 workgroups come of them: each segment
// reads the row's context again.
hipError_t launch_adjust(int type, AdjustArgs a, hipStream_t s) {
  if (a.R == 0) return hipSuccess;
  a.seg = 1024;
  while (a.seg < 8192 && a.R * ((a.V + a.seg - 1) / a.seg) > 2048) a.seg *= 2;
  a.segs = (int)(((long long)a.V + a.seg - 1) / a.seg);
  const size_t lds = a.ctx > 0 ? a.seg * sizeof(unsigned) : 0;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    LTC_LAUNCH((adjust_kernel<T>), dim3((unsigned)(a.R * a.segs)), dim3(kThreads), lds, s, a);
    return hipGetLastError();
  });
}

}  // namespace ltc
