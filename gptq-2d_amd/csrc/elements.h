// Element types of what callers pass beside fp32 and fp64 matrices (keys, values, queries, activations), and the operand
// types of the fp16 and bf16 matrix instructions.
#pragma once

#include "common.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

enum { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2 };

template <int TYPE>
struct Elem;
template <>
struct Elem<TYPE_F32> {
  typedef float T;
};
template <>
struct Elem<TYPE_BF16> {
  typedef uint16_t T;
};
template <>
struct Elem<TYPE_F16> {
  typedef _Float16 T;
};

template <int TYPE>
__device__ __forceinline__ float to_f32(typename Elem<TYPE>::T x) {
  if constexpr (TYPE == TYPE_BF16)
    return __uint_as_float((unsigned)x << 16);
  else
    return (float)x;
}
template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::T from_f32(float x) {
  if constexpr (TYPE == TYPE_BF16)
    return (uint16_t)(__float_as_uint(round_to_bf16(x)) >> 16);
  else
    return (typename Elem<TYPE>::T)x;
}

// N consecutive elements from p + d, 0 past `dim` (vector loads need only the element's own alignment).
template <int TYPE, int N>
__device__ __forceinline__ void load_row(float (&x)[N], const typename Elem<TYPE>::T* __restrict__ p, int d, int dim) {
  typedef typename Elem<TYPE>::T T;
  constexpr int V = 16 / (int)sizeof(T) < N ? 16 / (int)sizeof(T) : N;
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if (d + N <= dim) {
#pragma unroll
    for (int i = 0; i < N; i += V) {
      const vec v = *reinterpret_cast<const vec*>(p + d + i);
#pragma unroll
      for (int j = 0; j < V; ++j) x[i + j] = to_f32<TYPE>(v[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = d + i < dim ? to_f32<TYPE>(p[d + i]) : 0.f;
  }
}

// Eight consecutive elements as they lie, 0 past the row's end; loads only, so that several can be in flight.
template <int TYPE>
struct Raw8 {
  typedef typename Elem<TYPE>::T T;
  static constexpr int V = 16 / (int)sizeof(T);  // elements of a 16-byte load
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v[8 / V];
  __device__ __forceinline__ void load(const T* __restrict__ row, int d, int n) {
    if (d + 8 <= n) {
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) v[i] = *reinterpret_cast<const vec*>(row + d + V * i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i / V][i % V] = d + i < n ? row[d + i] : (T)0;
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32<TYPE>(v[i / V][i % V]); }
};

// Exponent e with 2^e <= x < 2^(e + 1) of a finite x > 0 (0 for anything else).
__device__ __forceinline__ int exponent_of(float x) {
  return x > 0.f && x < __builtin_inff() ? (int)__builtin_amdgcn_frexp_expf(x) - 1 : 0;
}

__device__ __forceinline__ half2v as_half2(unsigned u) { return __builtin_bit_cast(half2v, u); }
__device__ __forceinline__ half2v both(float x) { return (half2v){(_Float16)x, (_Float16)x}; }

// x & mask | 0x64006400 (two fp16 numbers of 1024 and up) in one instruction: with literals the compiler takes two, since
// an instruction holds one constant.
__device__ __forceinline__ half2v codes_at(unsigned x, unsigned mask) {
  unsigned r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(0x64006400u));
  return as_half2(r);
}

}  // namespace
