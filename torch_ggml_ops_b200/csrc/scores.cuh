// Rows of scores (a gate's or a head's logits) as the kernels of router.cu and logit_rules.cu read and
// write them: bf16, fp16 or fp32 in memory, fp32 in registers.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace tgo {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N elements that lie together, at their natural alignment of N * sizeof(T) <= 16 bytes
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

constexpr unsigned kAllLanes = 0xFFFFFFFFu;
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kAllLanes, v, d);
    return v;
}

// An unsigned number for every float, in the floats' order; -0 and +0 have the same.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order ^ (static_cast<uint32_t>(static_cast<int32_t>(~order) >> 31) | 0x80000000u));
}

}  // namespace tgo
