// A cache's values as floats.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace confkv {
namespace kv {

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

template <class T>
__device__ __forceinline__ T from_float(float x)
{
    if constexpr (std::is_same_v<T, float>) {
        return x;
    } else if constexpr (std::is_same_v<T, __half>) {
        return __float2half_rn(x);
    } else {
        return __float2bfloat16_rn(x);
    }
}

}  // namespace kv
}  // namespace confkv
