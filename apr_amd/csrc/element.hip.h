// element.hip.h -- the element types of the label operators (APR_F32, APR_F16, APR_BF16).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace apr {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, v) << 16); }
// one rounding to nearest even; beyond the type's range: infinity
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

}  // namespace apr
