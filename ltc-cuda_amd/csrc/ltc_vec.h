// Vectors of fp32, bf16 or fp16 values as the sequence and token kernels load, keep
// and store them.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

namespace ltc {

// V values of a type, kept packed in words of 32 bits.
template <class T, int V>
struct Vec {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  static_assert(kWords * 4 == V * (int)sizeof(T), "whole words");
  unsigned w[kWords];

  __device__ __forceinline__ float get(int v) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[v]);
    } else if constexpr (std::is_same<T, __bf16>::value) {
      return __uint_as_float(v & 1 ? w[v / 2] & 0xffff0000u : w[v / 2] << 16);
    } else {
      const unsigned short h = (unsigned short)(v & 1 ? w[v / 2] >> 16 : w[v / 2]);
      return (float)__builtin_bit_cast(_Float16, h);
    }
  }
  // The same for an index known at run time only. (A choice between the words
  // themselves becomes an indexed load, and the vector goes to scratch memory.)
  __device__ __forceinline__ float get_at(int i) const {
    constexpr int per = 4 / (int)sizeof(T);
    unsigned q = 0;
#pragma unroll
    for (int j = 0; j < kWords; ++j) q |= i / per == j ? w[j] : 0u;
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(q);
    } else {
      const unsigned short h = (unsigned short)(q >> (i & 1) * 16);
      return (float)__builtin_bit_cast(T, h);
    }
  }
  // Rounded to nearest, ties to even; the packed conversions take two.
  __device__ __forceinline__ void put(const float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int v = 0; v < V; ++v) w[v] = __float_as_uint(f[v]);
    } else {
      typedef float F2 __attribute__((ext_vector_type(2)));
      typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int v = 0; v < V; v += 2) {
        const F2 q = {f[v], f[v + 1]};
        w[v / 2] = __builtin_bit_cast(unsigned, __builtin_convertvector(q, T2));
      }
    }
  }
};

// n (< V: the row's last channels) of V values at p, which has T's alignment
// only: gfx950 takes wide global loads and stores at any address.
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p, int n) {
  Vec<T, V> r;
  if (n >= V) {
    __builtin_memcpy(r.w, p, sizeof(r.w));
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T, V>::kWords; ++i) r.w[i] = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < n) {
        if constexpr (sizeof(T) == 4) r.w[v] = reinterpret_cast<const unsigned*>(p)[v];
        else r.w[v / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[v] << (v & 1) * 16;
      }
  }
  return r;
}

template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& r, int n) {
  if (n >= V) {
    __builtin_memcpy(p, r.w, sizeof(r.w));
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < n) {
        if constexpr (sizeof(T) == 4) reinterpret_cast<unsigned*>(p)[v] = r.w[v];
        else reinterpret_cast<unsigned short*>(p)[v] = (unsigned short)(r.w[v / 2] >> (v & 1) * 16);
      }
  }
}

}  // namespace ltc
