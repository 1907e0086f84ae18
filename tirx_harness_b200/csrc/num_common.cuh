// Number formats and small numerics shared by the norm, routing and 4-bit kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "moe_ops.cuh"

namespace b200 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive values as they lie in memory: one 16-byte load for the 16-bit types, two for fp32.
template <typename T> struct alignas(16) Pack8 { T v[8]; };

template <typename T> __device__ __forceinline__ Pack8<T> load8(const T* p) {
    Pack8<T> r;
    const uint4* src = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) reinterpret_cast<uint4*>(&r)[i] = __ldg(src + i);
    return r;
}
// the same for data that is read once
template <typename T> __device__ __forceinline__ Pack8<T> load8_once(const T* p) {
    Pack8<T> r;
    const uint4* src = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) reinterpret_cast<uint4*>(&r)[i] = __ldcs(src + i);
    return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Pack8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// x / d, correctly rounded, for a divisor whose correctly rounded reciprocal r = 1 / d is at hand: q = x r, then one
// correction by the exact remainder (Markstein 1990: with r and the remainder correctly rounded the result is too).
// Needs d and 1/d normal and away from the ends of the range, which div_ok tests; a quotient whose remainder
// underflows is so small that every 8- or 4-bit format rounds it to zero either way.
__device__ __forceinline__ float div_by(float x, float d, float r) {
    const float q = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-d, q, x), r, q);
}
__device__ __forceinline__ bool div_ok(float d) { return d > 1e-30f && d < 1e30f; }

}  // namespace b200
