// Elements of 16 or 32 bits held in pairs as they lie in memory, and computed on as
// packed fp32 pairs (one instruction for two, sm100_ptx.cuh's f2_ functions): at 16 bits
// an element the arithmetic of a streaming kernel would otherwise take longer than its
// memory.
#pragma once

#include <type_traits>

#include "sm100_ptx.cuh"

namespace mgfa::dev {

template <class E>
__device__ __forceinline__ float to_f(E v);
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(float v) { return v; }

template <class E>
__device__ __forceinline__ E from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }

template <class E>
struct PairOf {
  using Raw = uint32_t;
  static __device__ __forceinline__ uint64_t wide(uint32_t r) {
    if constexpr (std::is_same_v<E, __nv_bfloat16>) {  // a bf16 is the upper half of its fp32
      return f2_pack(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    } else {
      const float2 f = unpack16<true>(r);
      return f2_pack(f.x, f.y);
    }
  }
  static __device__ __forceinline__ uint32_t narrow(uint64_t v) {
    float a, b;
    f2_unpack(v, a, b);
    return pack16<std::is_same_v<E, __half>>(a, b);
  }
};
template <>
struct PairOf<float> {
  using Raw = uint64_t;
  static __device__ __forceinline__ uint64_t wide(uint64_t r) { return r; }
  static __device__ __forceinline__ uint64_t narrow(uint64_t v) { return v; }
};

template <int kBytes>
struct Bytes;
template <>
struct Bytes<16> { using T = uint4; };
template <>
struct Bytes<8> { using T = uint2; };
template <>
struct Bytes<4> { using T = uint32_t; };
template <>
struct Bytes<2> { using T = uint16_t; };

}  // namespace mgfa::dev
