// f32, f16 and bf16 elements in the kernels of the 16-bit layers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace b200 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {  // (rounded to nearest even)
  if constexpr (sizeof(T) == 4) {
    return v;
  } else if constexpr (std::is_same<T, __half>::value) {
    return __float2half_rn(v);
  } else {
    return __float2bfloat16_rn(v);
  }
}

}  // namespace b200
