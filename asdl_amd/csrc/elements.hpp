// Element types of the operators that take fp32, bf16 and fp16 alike, loads of several of them at any alignment, and sums over a
// wave or a work group.  Arithmetic is fp32 or wider everywhere; a value is rounded once, when it is stored.
#pragma once
#include "common.hpp"

namespace ak {

template <typename T>
struct Type {
  using type = T;
};

// fn(Type<T>{}) for the element type of a dtype code; AK_ERR_ARG for a code that is none.
template <typename Fn>
inline int with_type(int dtype, Fn&& fn) {
  switch (dtype) {
    case AK_F32: return fn(Type<float>{});
    case AK_BF16: return fn(Type<__bf16>{});
    case AK_F16: return fn(Type<_Float16>{});
    default: return AK_ERR_ARG;
  }
}

inline bool is_element_type(int dtype) { return dtype == AK_F32 || dtype == AK_BF16 || dtype == AK_F16; }

// One element of a type known at run time (weights, biases: a few per lane).
__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == AK_F32) return static_cast<const float*>(p)[i];
  if (dtype == AK_BF16) return static_cast<float>(static_cast<const __bf16*>(p)[i]);
  return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}

__device__ __forceinline__ void store_from_float(void* p, int dtype, int64_t i, float v) {
  if (dtype == AK_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == AK_BF16) static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
  else static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The sum over a work group of WAVES waves, in every thread; `red` has WAVES words.  The barrier in front keeps the words of the
// sum before; the order of the sum is fixed.
template <int WAVES, typename V>
__device__ __forceinline__ V group_sum(V v, V* red) {
  v = wave_sum(v);
  if constexpr (WAVES == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V s = red[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += red[w];
  return s;
}

}  // namespace ak
