// Quantisation to 4-bit blocks (e2m1 codes under one scale per block), and the codes' values as e4m3.
//
//   nvfp4  16 values, scale s = e4m3(min(amax / (6 g), 448)) with one fp32 factor g: value = code * s * g
//   mxfp4  32 values, scale s = 2^(floor(log2 amax) - 2), at least 2^-127:           value = code * s
//   code = e2m1(x / (s g)), rounded to nearest with ties to even, magnitudes above 6 becoming 6
//
// A block that holds an infinity or a NaN gets the scale NaN and codes 0, so that it shows in every product with it.
//
// Codes are packed two to a byte, the earlier one in the low half.  Scales are stored in the order in which the tensor
// core takes them: tiles of 512 bytes for 128 rows x 4 blocks, row r's four bytes at (r % 32) * 16 + (r / 32) * 4; the
// tiles of a row block follow one another along K, which is filled up to a multiple of 256 with zero scales.
//
// Bound by memory.  A block of threads takes 128 rows x 256 columns, so that the scales it makes are whole tiles.
#pragma once

#include <cuda_fp4.h>

#include "num_common.cuh"

namespace b200 {

struct Fp4QuantParams {
    const void* x; long long x_stride;          // elements between rows
    const float* factor; int factor_stride;     // g of group i at factor[i * stride]; null: 1
    const int* src; int top_k;                  // row r comes from row src[r] / top_k; negative: r is left alone.  null: r
    uint8_t* q;
    uint8_t* sf;
    int rows;                                   // of one group
    int K;
    int gate_first;                             // SiLU*mul: which half of x is the gate
    int src_rows;                               // rows of x (of one group)
    int k_blocks;                               // 256-column pieces of K
};

// eight values -> eight codes, the first in the lowest four bits
__device__ __forceinline__ uint32_t pack8_e2m1(const float* v) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_E2M1, cudaRoundNearest) << (8 * i);
    return r;
}

constexpr int FP4_QUANT_THREADS = 256;

// NV: nvfp4, else mxfp4.  SILU: x holds gate and up, K columns each.
// A thread takes 16 columns of a row at a time (a block of nvfp4, half a block of mxfp4).
template <typename T, bool NV, bool SILU>
__global__ void __launch_bounds__(FP4_QUANT_THREADS) quant_fp4_kernel(const Fp4QuantParams p) {
    constexpr int WORDS = NV ? 4 : 2;           // scale tiles of 256 columns
    __shared__ uint32_t tile[WORDS * 128];
    const int group = blockIdx.y, row_blocks = (p.rows + 127) >> 7;
    const int rb = blockIdx.x / p.k_blocks, kb = blockIdx.x - rb * p.k_blocks;
    const int k0 = kb * 256, r0 = rb * 128;
    const int seg = threadIdx.x & 15, col = k0 + seg * 16;
    const float g = p.factor ? __ldg(p.factor + group * p.factor_stride) : 1.0f;
    const float g6 = __fmul_rn(6.0f, g);
    uint8_t* tb = reinterpret_cast<uint8_t*>(tile);
    const T* xg = static_cast<const T*>(p.x) + (long long)group * p.src_rows * p.x_stride;
#pragma unroll 2
    for (int i = threadIdx.x >> 4; i < 128; i += FP4_QUANT_THREADS / 16) {
        const int r = r0 + i;
        int s = r < p.rows ? r : -1;
        if (s >= 0 && p.src) { s = __ldg(p.src + r); if (s >= 0) s /= p.top_k; }
        const bool live = s >= 0 && s < p.src_rows && col < p.K;        // the same for all threads of a scale block
        float v[16];
        uint32_t amax = 0;
        if (live) {
            const T* row = xg + s * p.x_stride + col;
            const Pack8<T> a = load8(row + (SILU && !p.gate_first ? p.K : 0)), b = load8(row + (SILU && !p.gate_first ? p.K : 0) + 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) { v[j] = to_f32(a.v[j]); v[8 + j] = to_f32(b.v[j]); }
            if (SILU) {
                const Pack8<T> c = load8(row + (p.gate_first ? p.K : 0)), d = load8(row + (p.gate_first ? p.K : 0) + 8);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = __fmul_rn(silu_f32(v[j]), to_f32(c.v[j]));
                    v[8 + j] = __fmul_rn(silu_f32(v[8 + j]), to_f32(d.v[j]));
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
        if (!NV) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        uint32_t byte = 0, lo = 0, hi = 0;
        if (live) {
            const bool finite = amax < 0x7F800000u;
            if (NV) {
                const float t = fminf(__fdiv_rn(__uint_as_float(amax), g6), 448.0f);
                byte = finite ? __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3) : 0x7Fu;
                const float unit = __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3))), g);
                if (finite && unit > 0.0f) {
                    if (div_ok(unit)) {
                        const float rc = __frcp_rn(unit);
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = div_by(v[j], unit, rc);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = __fdiv_rn(v[j], unit);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = 0.0f;
                }
            } else {
                const int e = (int)(amax >> 23) - 2;
                byte = finite ? (uint32_t)max(e, 0) : 0xFFu;
                const float inv = finite ? __uint_as_float((254u - byte) << 23) : 0.0f;         // 2^(127 - byte), exact
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = finite ? __fmul_rn(v[j], inv) : 0.0f;
            }
            lo = pack8_e2m1(v);
            hi = pack8_e2m1(v + 8);
            *reinterpret_cast<uint2*>(p.q + ((long long)group * p.rows + r) * (p.K >> 1) + (col >> 1)) = make_uint2(lo, hi);
        }
        const int b = NV ? seg : seg >> 1;                  // block of these 256 columns
        if (NV || !(seg & 1)) tb[(b >> 2) * 512 + (i & 31) * 16 + (i >> 5) * 4 + (b & 3)] = (uint8_t)byte;
    }
    __syncthreads();
    uint32_t* out = reinterpret_cast<uint32_t*>(p.sf) + (((long long)group * row_blocks + rb) * p.k_blocks + kb) * (WORDS * 128);
    for (int w = threadIdx.x; w < WORDS * 128; w += FP4_QUANT_THREADS) {
        const int r = r0 + ((w & 127) >> 2) + (w & 3) * 32;
        // rows that are left alone keep their scales; those behind the last one are zero
        if (p.src == nullptr || r >= p.rows || __ldg(p.src + r) >= 0) out[w] = tile[w];
    }
}

// Packed codes -> e4m3 values, 16 per thread.
__global__ void __launch_bounds__(256) unpack_fp4_kernel(const uint2* __restrict__ q, uint4* __restrict__ out, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint2 w = __ldcs(q + i);
    // magnitudes 0 .5 1 1.5 | 2 3 4 6 as e4m3 bytes; a code's low three bits pick one, its fourth is the sign
    auto four = [](uint32_t c) {
        const uint32_t mag = __byte_perm(0x3C383000u, 0x4C484440u, c & 0x7777u);
        const uint32_t sign = ((c & 0x8u) << 4) | ((c & 0x80u) << 8) | ((c & 0x800u) << 12) | ((c & 0x8000u) << 16);
        return mag | sign;
    };
    __stcs(out + i, make_uint4(four(w.x & 0xFFFFu), four(w.x >> 16), four(w.y & 0xFFFFu), four(w.y >> 16)));
}

}  // namespace b200
