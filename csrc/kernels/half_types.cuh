// The two 16-bit operand types (bf16, fp16): packing, unpacking and the tcgen05 operand format code.
#pragma once
#include "common.cuh"

namespace br {

template <typename T>
struct Half16;

template <>
struct Half16<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;  // instruction descriptor's operand format: bf16
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return unpack_bf16(u); }
};

template <>
struct Half16<__half> {
  static constexpr uint32_t kFormat = 0;  // fp16
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    __half2 v = *reinterpret_cast<__half2*>(&u);
    return __half22float2(v);
  }
};

}  // namespace br
