// Root-mean-square norm of the residual stream with an 8-bit output, and its gradient.
//
// forward, one row:   h = round(x + residual)              (in the inputs' type: the stream the next layer reads)
//                     rstd = (sum h^2 / H + eps) ^ -1/2     y = h * rstd * w
//                     per 128 columns: s = max(amax|y|, 1e-8) / 448 (or that, rounded up to a power of two), q = e4m3(y / s)
// gradient, one row:  g = dy * w,  dx = rstd * g - h * rstd^3 / H * sum(g h)  (+ dh),  dw = sum over rows of dy * h * rstd
//
// Both are bound by memory: a row is read once, held in registers between the sum and the output, and written once.
// Every sum is kept in fp32.
#pragma once

#include "num_common.cuh"

namespace b200 {

struct NormParams {
    const void* x; long long x_stride;
    const void* residual; long long res_stride;
    const void* weight;
    uint8_t* q;
    float* scales; long long ss_row, ss_blk;
    void* h;                   // written where a residual is added
    void* y;                   // may be null
    float* rstd;
    int T, H;
    float eps;
    int pow2;
};

// Sum over the block; every thread gets it.  `buf` holds 33 floats.
__device__ __forceinline__ float block_sum(float v, float* buf) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    // every warp adds the partial sums up for itself, in the same order: one barrier instead of two
    float s = lane < warps ? buf[lane] : 0.0f;
    return warp_sum(s);
}

constexpr int NORM_MAX_THREADS = 512;
constexpr int NORM_MAX_H = 512 * 4 * 8;        // four pieces of 8 columns per thread
constexpr int NORM_GRAD_MAX_PARTS = 512;

// One block per row; thread t holds the 8-column pieces t, t + blockDim, ... (CH of them).  A 128-column block is 16
// neighbouring threads of one piece, so its largest value takes four shuffles.
template <typename T, typename W, int CH>
__global__ void __launch_bounds__(NORM_MAX_THREADS) rms_norm_quant_kernel(const NormParams p) {
    __shared__ float buf[32];
    const int row = blockIdx.x, n8 = p.H >> 3;
    const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* rr = p.residual ? static_cast<const T*>(p.residual) + row * p.res_stride : nullptr;
    Pack8<T> xv[CH], rv[CH];
    Pack8<W> wv[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i < n8) {
            xv[c] = load8_once(xr + i * 8);
            if (rr) rv[c] = load8_once(rr + i * 8);
            wv[c] = load8(static_cast<const W*>(p.weight) + i * 8);
        }
    }
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i < n8) {
            if (rr) {
#pragma unroll
                for (int j = 0; j < 8; ++j) xv[c].v[j] = from_f32<T>(to_f32(xv[c].v[j]) + to_f32(rv[c].v[j]));
                store8(static_cast<T*>(p.h) + (long long)row * p.H + i * 8, xv[c]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) { const float f = to_f32(xv[c].v[j]); sq = fmaf(f, f, sq); }
        }
    }
    const float rstd = __frsqrt_rn(__fdiv_rn(block_sum(sq, buf), (float)p.H) + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        float y[8];
        uint32_t amax = 0;                  // largest magnitude as bits: infinities and NaN order above every number
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[j] = i < n8 ? __fmul_rn(__fmul_rn(to_f32(xv[c].v[j]), rstd), to_f32(wv[c].v[j])) : 0.0f;
            amax = max(amax, __float_as_uint(y[j]) & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (i >= n8) continue;              // no shuffle below
        const float a = __uint_as_float(amax);
        float s = __fdiv_rn(a < 1.0e-8f ? 1.0e-8f : a, 448.0f);          // a NaN stays one
        if (p.pow2 && s < INFINITY) {
            const uint32_t b = __float_as_uint(s);
            s = __uint_as_float((b + 0x7FFFFFu) & 0xFF800000u);          // up to the next power of two
        }
        uint2 q;
        if (div_ok(s)) {
            const float r = __frcp_rn(s);
            q.x = pack4_e4m3(div_by(y[0], s, r), div_by(y[1], s, r), div_by(y[2], s, r), div_by(y[3], s, r));
            q.y = pack4_e4m3(div_by(y[4], s, r), div_by(y[5], s, r), div_by(y[6], s, r), div_by(y[7], s, r));
        } else {
            q.x = pack4_e4m3(__fdiv_rn(y[0], s), __fdiv_rn(y[1], s), __fdiv_rn(y[2], s), __fdiv_rn(y[3], s));
            q.y = pack4_e4m3(__fdiv_rn(y[4], s), __fdiv_rn(y[5], s), __fdiv_rn(y[6], s), __fdiv_rn(y[7], s));
        }
        *reinterpret_cast<uint2*>(p.q + (long long)row * p.H + i * 8) = q;
        if ((i & 15) == 0) p.scales[row * p.ss_row + (i >> 4) * p.ss_blk] = s;
        if (p.y) {
            Pack8<T> o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o.v[j] = from_f32<T>(y[j]);
            store8(static_cast<T*>(p.y) + (long long)row * p.H + i * 8, o);
        }
    }
}

struct NormGradParams {
    const void* dy; long long dy_stride;
    const void* h; long long h_stride;
    const void* weight;
    const float* rstd;
    const void* dh; long long dh_stride;      // gradient that reaches h past the norm; may be null
    void* dx;
    float* partial;                           // [gridDim.x, H]: each block's share of dw
    int T, H;
};

// Blocks walk the rows with a stride; a thread keeps its columns' share of dw in registers all the while, so dw costs
// one row of fp32 per block instead of a second pass over dy and h.
template <typename T, typename W, int CH>
__global__ void __launch_bounds__(NORM_MAX_THREADS) rms_norm_grad_kernel(const NormGradParams p) {
    __shared__ float buf[2][32];
    const int n8 = p.H >> 3;
    float dw[CH][8];
    Pack8<W> wv[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[c][j] = 0.0f;
        if (i < n8) wv[c] = load8(static_cast<const W*>(p.weight) + i * 8);
    }
    int flip = 0;                             // two buffers: one barrier per row is enough
    for (int row = blockIdx.x; row < p.T; row += gridDim.x, flip ^= 1) {
        const T* dyr = static_cast<const T*>(p.dy) + row * p.dy_stride;
        const T* hr = static_cast<const T*>(p.h) + row * p.h_stride;
        const T* dhr = p.dh ? static_cast<const T*>(p.dh) + row * p.dh_stride : nullptr;
        Pack8<T> dyv[CH], hv[CH], dv[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
            if (i < n8) {
                dyv[c] = load8_once(dyr + i * 8);
                hv[c] = load8_once(hr + i * 8);
                if (dhr) dv[c] = load8_once(dhr + i * 8);
            }
        }
        const float rstd = __ldg(p.rstd + row);
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
            if (i < n8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = to_f32(dyv[c].v[j]), n = to_f32(hv[c].v[j]) * rstd;
                    dw[c][j] = fmaf(d, n, dw[c][j]);
                    dot = fmaf(d * to_f32(wv[c].v[j]), n, dot);
                }
            }
        }
        const float mean = __fdiv_rn(block_sum(dot, buf[flip]), (float)p.H);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
            if (i < n8) {
                Pack8<T> o;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float g = to_f32(dyv[c].v[j]) * to_f32(wv[c].v[j]), n = to_f32(hv[c].v[j]) * rstd;
                    float v = rstd * fmaf(-n, mean, g);
                    if (dhr) v += to_f32(dv[c].v[j]);
                    o.v[j] = from_f32<T>(v);
                }
                store8(static_cast<T*>(p.dx) + (long long)row * p.H + i * 8, o);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i < n8) {
            float4* dst = reinterpret_cast<float4*>(p.partial + (long long)blockIdx.x * p.H + i * 8);
            dst[0] = make_float4(dw[c][0], dw[c][1], dw[c][2], dw[c][3]);
            dst[1] = make_float4(dw[c][4], dw[c][5], dw[c][6], dw[c][7]);
        }
    }
}

// dw[c] = sum of the blocks' shares, always in the same order.  Block: 32 columns x 32 strands of blocks.
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* __restrict__ partial, float* __restrict__ dw, int parts, int H) {
    __shared__ float t[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < H)
        for (int i = strand; i < parts; i += 32) s += __ldg(partial + (long long)i * H + c);
    t[strand][threadIdx.x & 31] = s;
    __syncthreads();
    s = warp_sum(t[threadIdx.x & 31][strand]);
    const int col = blockIdx.x * 32 + strand;
    if ((threadIdx.x & 31) == 0 && col < H) dw[col] = s;
}

}  // namespace b200
