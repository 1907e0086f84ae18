// m-grouped GEMM of 4-bit block-scaled operands: D_g = alpha_g * deq(A_g) * deq(B_g)^T.
#pragma once

#include "fp4_ops.cuh"

namespace b200 {

struct GGFp4Params {
    const uint8_t *a, *b, *sfa, *sfb;
    const float* alpha; int alpha_stride;       // null: 1
    const int* layout;
    const int* rows_used;
    void* d; long long ldd; int d_f32;
    int G, M, N, K, masked;
    int kt;                                     // scale tiles along K
    int a_tiles, b_tiles;                       // 128-row scale blocks of a (one group of the masked layout) and of one b
};

__device__ __forceinline__ float fp4_scale(const uint8_t* tiles, long long block128, int kt, int row, int blk, bool nv) {
    const uint8_t byte = __ldg(tiles + (block128 * kt + (blk >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (blk & 3));
    if (nv) return __half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3)));
    return byte == 255 ? NAN : byte == 0 ? __uint_as_float(1u << 22) : __uint_as_float((uint32_t)byte << 23);
}
__device__ __forceinline__ float fp4_code(uint32_t c) {
    const float v[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
    const float x = v[c & 7u];
    return (c & 8u) ? -x : x;
}

// 64 x 64 tile, 16 x 16 threads of 4 x 4 outputs; 32 values of K at a time, dequantised into shared memory.
template <bool NV>
__global__ void __launch_bounds__(256) gg_fp4_simple_kernel(const GGFp4Params p) {
    __shared__ float sa[32][65], sb[32][65];
    const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    constexpr int BLK = NV ? 16 : 32;
    int row_end = p.M;
    if (!p.masked && p.rows_used) row_end = min(p.M, max(0, __ldg(p.rows_used)));
    int group = p.masked ? (int)blockIdx.z : -1;
    while (true) {
        if (p.masked) row_end = min(p.M, max(0, __ldg(p.layout + group)));
        else {
            // the next group that has rows here
            int best = p.G;
            for (int i = 0; i < 64; ++i)
                if (m0 + i < row_end) {
                    const int g = __ldg(p.layout + m0 + i);
                    if (g > group && g < best) best = g;
                }
            if (best >= p.G) return;
            group = best;
        }
        if (m0 >= row_end) return;
        float acc[4][4] = {};
        const long long arow0 = p.masked ? (long long)group * p.M : 0;
        for (int k0 = 0; k0 < p.K; k0 += 32) {
            __syncthreads();
            for (int i = threadIdx.x; i < 64 * 16; i += 256) {
                const int r = i >> 4, kb = i & 15, k = k0 + kb * 2;
                float x0 = 0, x1 = 0, y0 = 0, y1 = 0;
                if (m0 + r < row_end) {
                    const uint8_t c = __ldg(p.a + (arow0 + m0 + r) * (p.K / 2) + k / 2);
                    const int lr = m0 + r;
                    const long long tb = (p.masked ? (long long)group * p.a_tiles : 0) + (lr >> 7);
                    const float s = fp4_scale(p.sfa, tb, p.kt, lr & 127, k / BLK, NV);
                    x0 = fp4_code(c & 15) * s; x1 = fp4_code(c >> 4) * s;
                }
                if (n0 + r < p.N) {
                    const uint8_t c = __ldg(p.b + ((long long)group * p.N + n0 + r) * (p.K / 2) + k / 2);
                    const int n = n0 + r;
                    const float s = fp4_scale(p.sfb, (long long)group * p.b_tiles + (n >> 7), p.kt, n & 127, k / BLK, NV);
                    y0 = fp4_code(c & 15) * s; y1 = fp4_code(c >> 4) * s;
                }
                sa[kb * 2][r] = x0; sa[kb * 2 + 1][r] = x1;
                sb[kb * 2][r] = y0; sb[kb * 2 + 1][r] = y1;
            }
            __syncthreads();
#pragma unroll 8
            for (int k = 0; k < 32; ++k) {
                float x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[i] = sa[k][ty + 16 * i]; y[i] = sb[k][tx + 16 * i]; }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
            }
        }
        const float al = p.alpha ? __ldg(p.alpha + group * p.alpha_stride) : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (r >= row_end || n >= p.N) continue;
                if (!p.masked && __ldg(p.layout + r) != group) continue;
                const long long o = (arow0 + r) * p.ldd + n;
                const float v = acc[i][j] * al;
                if (p.d_f32) static_cast<float*>(p.d)[o] = v;
                else static_cast<__nv_bfloat16*>(p.d)[o] = __float2bfloat16_rn(v);
            }
        if (p.masked) return;
    }
}

}  // namespace b200
