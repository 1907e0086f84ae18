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

// Pairs of fp32 values: sm_100 adds, multiplies and multiply-adds two at a time, each rounded as the single one is.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f32x2 both(float v) { return pack_f32x2(v, v); }
__device__ __forceinline__ float lo2(f32x2 v) { float a, b; unpack_f32x2(v, a, b); return a; }
__device__ __forceinline__ float hi2(f32x2 v) { float a, b; unpack_f32x2(v, a, b); return b; }

// Eight consecutive values of type T as they lie in memory (16 bytes, fp32: 32), and the same as four fp32 pairs.
template <typename T> struct alignas(16) Raw8 { uint4 w[sizeof(T) / 2]; };
template <typename T> struct Fmt;
template <> struct Fmt<__nv_bfloat16> {
    static __device__ __forceinline__ f32x2 up(uint32_t u) { return pack_f32x2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t down(f32x2 v) { return cvt_bf16x2(v); }
};
template <> struct Fmt<__half> {
    static __device__ __forceinline__ f32x2 up(uint32_t u) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        return pack_f32x2(f.x, f.y);
    }
    static __device__ __forceinline__ uint32_t down(f32x2 v) {
        const __half2 h = __floats2half2_rn(lo2(v), hi2(v));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <typename T> __device__ __forceinline__ void unpack8(const Raw8<T>& r, f32x2 (&v)[4]) {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = Fmt<T>::up(u[i]);
}
template <> __device__ __forceinline__ void unpack8<float>(const Raw8<float>& r, f32x2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[2 * i] = pack_f32x2(__uint_as_float(r.w[i].x), __uint_as_float(r.w[i].y));
        v[2 * i + 1] = pack_f32x2(__uint_as_float(r.w[i].z), __uint_as_float(r.w[i].w));
    }
}
// rounded to T
template <typename T> __device__ __forceinline__ Raw8<T> pack8(const f32x2 (&v)[4]) {
    Raw8<T> r;
    r.w[0] = make_uint4(Fmt<T>::down(v[0]), Fmt<T>::down(v[1]), Fmt<T>::down(v[2]), Fmt<T>::down(v[3]));
    return r;
}
template <> __device__ __forceinline__ Raw8<float> pack8<float>(const f32x2 (&v)[4]) {
    Raw8<float> r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        r.w[i] = make_uint4(__float_as_uint(lo2(v[2 * i])), __float_as_uint(hi2(v[2 * i])), __float_as_uint(lo2(v[2 * i + 1])), __float_as_uint(hi2(v[2 * i + 1])));
    return r;
}
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return r;
}
template <typename T> __device__ __forceinline__ Raw8<T> lds8(const T* p) {          // shared memory
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

// the same for data that is not wanted in the L2 cache any longer
template <typename T> __device__ __forceinline__ void store8_streaming(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) __stcs(reinterpret_cast<uint4*>(p) + i, r.w[i]);
}

// the larger magnitude; a NaN stays one
__device__ __forceinline__ float amax_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

// contiguous global -> shared copy, completion on an mbarrier; both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// the same; the lines read are the first to leave the L2 cache
__device__ __forceinline__ void bulk_load_once(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t bar) {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
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
__device__ __forceinline__ f32x2 div_by(f32x2 x, f32x2 minus_d, f32x2 r) {
    const f32x2 q = mul2(x, r);
    return fma2(fma2(minus_d, q, x), r, q);
}
__device__ __forceinline__ bool div_ok(float d) { return d > 1e-30f && d < 1e30f; }
// x / d for four pairs
__device__ __forceinline__ void div8(f32x2 (&v)[4], float d) {
    if (div_ok(d)) {
        const f32x2 r = both(__frcp_rn(d)), m = both(-d);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = div_by(v[i], m, r);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pack_f32x2(__fdiv_rn(lo2(v[i]), d), __fdiv_rn(hi2(v[i]), d));
    }
}
// eight values -> e4m3 bytes
__device__ __forceinline__ uint2 pack8_e4m3(const f32x2 (&v)[4]) {
    return make_uint2(pack4_e4m3(lo2(v[0]), hi2(v[0]), lo2(v[1]), hi2(v[1])), pack4_e4m3(lo2(v[2]), hi2(v[2]), lo2(v[3]), hi2(v[3])));
}

}  // namespace b200
