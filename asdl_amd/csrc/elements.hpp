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

// N neighbouring elements on their way, at any alignment (unaligned 16-byte loads and stores are one instruction).
template <typename T, int N>
struct Some {
  typedef T vec __attribute__((ext_vector_type(N)));
  vec v;
  __device__ __forceinline__ void load(const T* __restrict__ p) { __builtin_memcpy(&v, p, sizeof(T) * N); }
  __device__ __forceinline__ void clear() { v = vec{}; }
  __device__ __forceinline__ float get(int e) const { return static_cast<float>(v[e]); }
  __device__ __forceinline__ void set(int e, float x) { v[e] = static_cast<T>(x); }
  __device__ __forceinline__ void store(T* __restrict__ p) const { __builtin_memcpy(p, &v, sizeof(T) * N); }
};

// v + v of the lane that a data-parallel-primitive control selects.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// The sum over L = 16 or 64 neighbouring lanes, in each of them: swaps of neighbours, of pairs, mirrored halves and rows of 16 (moves
// between lanes as operands of the addition, where __shfl_xor goes through the LDS six times), then the four rows of a wave.
template <int L = 64>
__device__ __forceinline__ float lanes_sum(float v) {
  v = add_dpp<0xB1>(v);          // quad_perm 1 0 3 2
  v = add_dpp<0x4E>(v);          // quad_perm 2 3 0 1
  v = add_dpp<0x141>(v);         // row_half_mirror
  v = add_dpp<0x140>(v);         // row_mirror
  if constexpr (L == 64) {
    const int b = __builtin_bit_cast(int, v);
    const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 0)), r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 16));
    const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 32)), r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(b, 48));
    v = (r0 + r1) + (r2 + r3);
  }
  return v;
}

typedef unsigned long long u64;

template <int CTRL>
__device__ __forceinline__ u64 add_dpp(u64 v) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, 0xf, 0xf, true));
  return v + (static_cast<u64>(hi) << 32 | lo);
}

__device__ __forceinline__ u64 read_lane(u64 v, int lane) {
  return static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <>
__device__ __forceinline__ float wave_sum<float>(float v) {
  return lanes_sum<64>(v);
}
template <>
__device__ __forceinline__ u64 wave_sum<u64>(u64 v) {
  v = add_dpp<0xB1>(v);
  v = add_dpp<0x4E>(v);
  v = add_dpp<0x141>(v);
  v = add_dpp<0x140>(v);
  return (read_lane(v, 0) + read_lane(v, 16)) + (read_lane(v, 32) + read_lane(v, 48));
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
