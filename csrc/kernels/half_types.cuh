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

// Instruction descriptor for kind::f16 with both operands of type T and f32 accumulation.
template <typename T>
__host__ __device__ constexpr uint32_t umma_idesc_16(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (Half16<T>::kFormat << 7) | (Half16<T>::kFormat << 10) | (static_cast<uint32_t>(a_mn) << 15) |
         (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

}  // namespace br
