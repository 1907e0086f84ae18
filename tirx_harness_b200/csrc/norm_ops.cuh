// Root-mean-square norm of the residual stream with an 8-bit output, and its gradient.
//
// forward, one row:   h = round(x + residual)              (in the inputs' type: the stream the next layer reads)
//                     rstd = (sum h^2 / H + eps) ^ -1/2     y = h * rstd * w
//                     per 128 columns: s = max(amax|y|, 1e-8) / 448 (or that, rounded up to a power of two), q = e4m3(y / s)
// gradient, one row:  g = dy * w,  dx = rstd * (g - n * mean(g n)) (+ dh),  n = h * rstd;  dw = sum over rows of dy * n
//
// Both are bound by memory: a row is read once, held in registers between the sum and the output, and written once.  What
// keeps memory busy is the number of rows under way, not the number of threads: blocks stay on their SM and walk the rows
// with a stride, and bulk copies bring the next rows into a ring in shared memory while the current one is worked on
// (16384 x 7168 bf16 forward: 131 us, 6.3 TB/s; one row per block and its loads in registers: 205 us).
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
    int stages;                // rows of the ring
    int* status;
};

constexpr int NORM_MAX_THREADS = 512;
constexpr int NORM_MAX_H = 512 * 4 * 8;        // four pieces of 8 columns per thread
constexpr int NORM_MAX_STAGES = 4;
constexpr int NORM_HEAD_BYTES = 512;           // shared memory in front of the ring: barriers, flags, from 128 on the sums

// The ring of rows: `streams` inputs of `row_bytes` each per stage.  Thread 0 issues, everybody waits.
struct RowRing {
    uint64_t* full;
    uint8_t* data;
    volatile int* abort_flag;
    int* status;
    int stages, row_bytes, streams;
    int stage = 0;
    uint32_t phase = 0;
    bool live = true;

    __device__ __forceinline__ RowRing(uint8_t* smem, int stages_, int row_bytes_, int streams_, int* status_)
        : full(reinterpret_cast<uint64_t*>(smem)), data(smem + NORM_HEAD_BYTES),
          abort_flag(reinterpret_cast<volatile int*>(smem + 64)), status(status_), stages(stages_), row_bytes(row_bytes_), streams(streams_) {
        if (threadIdx.x == 0) {
            for (int s = 0; s < stages; ++s) mbar_init(smem_u32(full + s), 1);
            *abort_flag = 0;
            fence_mbar_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ uint8_t* at(int s, int stream) const { return data + (s * streams + stream) * row_bytes; }
    __device__ __forceinline__ void expect(int s) const { mbar_arrive_expect_tx(smem_u32(full + s), row_bytes * streams); }
    __device__ __forceinline__ void load(int s, int stream, const void* src) const {
        bulk_load(smem_u32(at(s, stream)), src, row_bytes, smem_u32(full + s));
    }
    __device__ __forceinline__ void load_once(int s, int stream, const void* src) const {
        bulk_load_once(smem_u32(at(s, stream)), src, row_bytes, smem_u32(full + s));
    }
    // A wait that runs out sets the status word; this row and those behind it are then made of whatever the stages hold, thread 0
    // issues no further copies, and those in flight get time to land before the block's memory goes (leave).
    __device__ __forceinline__ void wait() { live = mbar_wait_warp(smem_u32(full + stage), phase, abort_flag, status, STATUS_TIMEOUT_SMEM_FULL) && live; }
    __device__ __forceinline__ void leave() const {
        if (threadIdx.x == 0 && !live) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {}
        }
    }
    __device__ __forceinline__ void next() { if (++stage == stages) { stage = 0; phase ^= 1; } }
};

// Sum over the block; every thread gets it.  One barrier: two buffers used in turn keep the next sum's writes from this one's reads.
__device__ __forceinline__ float block_sum(float v, float* buf) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    return warp_sum(lane < warps ? buf[lane] : 0.0f);          // every warp for itself, in the same order
}

// Piece i of row `row` of y: the scale of its 128 columns from its largest magnitude, and y, scale and codes are stored.  All threads
// of a warp take part; pieces from H / 8 on have amax 0 and are not stored.
template <typename T>
__device__ __forceinline__ void norm_put(const NormParams& p, int row, int i, float amax, f32x2 (&y)[4]) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (i < (p.H >> 3)) {
        float s = __fdiv_rn(amax < 1.0e-8f ? 1.0e-8f : amax, 448.0f);          // a NaN stays one
        if (p.pow2 && s < INFINITY) s = __uint_as_float((__float_as_uint(s) + 0x7FFFFFu) & 0xFF800000u);     // up to the next power of two
        if ((i & 15) == 0) p.scales[row * p.ss_row + (i >> 4) * p.ss_blk] = s;
        if (p.y) store8(static_cast<T*>(p.y) + (long long)row * p.H + i * 8, pack8<T>(y));
        div8(y, s);
        *reinterpret_cast<uint2*>(p.q + (long long)row * p.H + i * 8) = pack8_e4m3(y);
    }
}

// The rows of this block whose squares pass fp32's range (rstd is 0) once more, in units of 2^72; a row with an infinity comes out
// as it was.  Called by the whole block behind its loop, whose registers and time it leaves alone (16384 x 7168: 130 us; inside the
// loop 137 us).
template <typename T, typename W>
__device__ __noinline__ void rms_norm_again(const NormParams p, float* sums) {
    constexpr float unit = 0x1p-72f;
    const int n8 = p.H >> 3, step = gridDim.x;
    auto load = [&](int row, int i, f32x2 (&h)[4]) {
        unpack8(load8(static_cast<const T*>(p.x) + row * p.x_stride + i * 8), h);
        if (!p.residual) return;
        f32x2 r[4];
        unpack8(load8(static_cast<const T*>(p.residual) + row * p.res_stride + i * 8), r);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = add2(h[j], r[j]);
        unpack8(pack8<T>(h), h);
    };
    __syncthreads();
    for (int row = blockIdx.x;; row += step) {
        if (*static_cast<volatile const float*>(p.rstd + row) == 0.0f) {          // the same for all threads
            f32x2 sq = 0, h[4];
            for (int i = threadIdx.x; i < n8; i += blockDim.x) {
                load(row, i, h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    h[j] = mul2(h[j], both(unit));
                    sq = fma2(h[j], h[j], sq);
                }
            }
            const float total = block_sum(lo2(sq) + hi2(sq), sums);
            const float rstd = __frsqrt_rn(__fdiv_rn(total, (float)p.H) + p.eps * unit * unit) * unit;
            if (threadIdx.x == 0) p.rstd[row] = rstd;
            for (int base = 0; base < n8; base += blockDim.x) {
                const int i = base + threadIdx.x;
                float amax = 0.0f;
                if (i < n8) {
                    f32x2 w[4];
                    load(row, i, h);
                    unpack8(load8(static_cast<const W*>(p.weight) + i * 8), w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        h[j] = mul2(mul2(h[j], both(rstd)), w[j]);
                        amax = amax_nan(amax_nan(amax, lo2(h[j])), hi2(h[j]));
                    }
                }
                norm_put<T>(p, row, i, amax, h);
            }
            __syncthreads();                   // the sums have been read
        }
        if (p.T - row <= step) break;
    }
}

// Thread t holds the 8-column pieces t, t + blockDim, ... (CH of them).  A 128-column block is 16 neighbouring threads of
// one piece, so its largest value takes four shuffles.
template <typename T, typename W, int CH>
__global__ void __launch_bounds__(NORM_MAX_THREADS) rms_norm_quant_kernel(const NormParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    float* sums = reinterpret_cast<float*>(smem + 128);
    volatile int* past = reinterpret_cast<volatile int*>(smem + 96);          // a sum of squares was infinite
    if (threadIdx.x == 0) *past = 0;
    const int n8 = p.H >> 3, step = gridDim.x;
    const bool res = p.residual != nullptr;
    RowRing ring(smem, p.stages, p.H * (int)sizeof(T), res ? 2 : 1, p.status);
    auto fetch = [&](int s, int row) {
        ring.expect(s);
        ring.load(s, 0, static_cast<const T*>(p.x) + row * p.x_stride);
        if (res) ring.load(s, 1, static_cast<const T*>(p.residual) + row * p.res_stride);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < p.stages && (long long)blockIdx.x + (long long)s * step < p.T; ++s) fetch(s, blockIdx.x + s * step);
    Raw8<W> wv[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i < n8) wv[c] = load8(static_cast<const W*>(p.weight) + i * 8);
    }
    int flip = 0;
    for (int row = blockIdx.x; row < p.T; flip ^= 32) {
        ring.wait();
        f32x2 h[CH][4];
        f32x2 sq = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) h[c][j] = 0;
            if (i < n8) {
                unpack8(lds8(reinterpret_cast<const T*>(ring.at(ring.stage, 0)) + i * 8), h[c]);
                if (res) {
                    f32x2 r[4];
                    unpack8(lds8(reinterpret_cast<const T*>(ring.at(ring.stage, 1)) + i * 8), r);
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[c][j] = add2(h[c][j], r[j]);
                    const Raw8<T> o = pack8<T>(h[c]);
                    store8(static_cast<T*>(p.h) + (long long)row * p.H + i * 8, o);
                    unpack8(o, h[c]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sq = fma2(h[c][j], h[c][j], sq);
            }
        }
        const float total = block_sum(lo2(sq) + hi2(sq), sums + flip);
        // the stage has been read by every thread: it can take the row after those under way
        const long long ahead = (long long)row + (long long)p.stages * step;
        if (threadIdx.x == 0 && ring.live && ahead < p.T) fetch(ring.stage, (int)ahead);
        ring.next();
        const float rstd = __frsqrt_rn(__fdiv_rn(total, (float)p.H) + p.eps);
        if (threadIdx.x == 0) {
            p.rstd[row] = rstd;
            if (rstd == 0.0f) *past = 1;
        }
        const f32x2 rstd2 = both(rstd);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
            f32x2 w[4];
            unpack8(wv[c], w);
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[c][j] = i < n8 ? mul2(mul2(h[c][j], rstd2), w[j]) : 0;
                amax = amax_nan(amax_nan(amax, lo2(h[c][j])), hi2(h[c][j]));
            }
            norm_put<T>(p, row, i, amax, h[c]);
        }
        if (p.T - row <= step) break;          // row + step could pass 2^31
        row += step;
    }
    ring.leave();
    __syncthreads();
    if (*past) rms_norm_again<T, W>(p, sums);
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
    int stages;
    int* status;
};

// A thread keeps its columns' share of dw in registers over all rows of its block, so dw costs one row of fp32 per block
// instead of a second pass over dy and h.  Inputs and dx pass through the L2 cache as data that is not read again: 8192 x 7168
// bf16 80 us (5.8 TB/s) instead of 87 us; the same costs the forward pass 5 to 15 %.
template <typename T, typename W, int CH>
__global__ void __launch_bounds__(NORM_MAX_THREADS) rms_norm_grad_kernel(const NormGradParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    float* sums = reinterpret_cast<float*>(smem + 128);
    const int n8 = p.H >> 3, step = gridDim.x;
    const bool past = p.dh != nullptr;
    RowRing ring(smem, p.stages, p.H * (int)sizeof(T), past ? 3 : 2, p.status);
    auto fetch = [&](int s, int row) {
        ring.expect(s);
        ring.load_once(s, 0, static_cast<const T*>(p.dy) + row * p.dy_stride);
        ring.load_once(s, 1, static_cast<const T*>(p.h) + row * p.h_stride);
        if (past) ring.load_once(s, 2, static_cast<const T*>(p.dh) + row * p.dh_stride);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < p.stages && (long long)blockIdx.x + (long long)s * step < p.T; ++s) fetch(s, blockIdx.x + s * step);
    f32x2 dw[CH][4];
    Raw8<W> wv[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) dw[c][j] = 0;
        if (i < n8) wv[c] = load8(static_cast<const W*>(p.weight) + i * 8);
    }
    int flip = 0;
    for (int row = blockIdx.x; row < p.T; flip ^= 32) {
        const float rstd = __ldg(p.rstd + row);
        const f32x2 rstd2 = both(rstd);
        ring.wait();
        Raw8<T> dyv[CH], hv[CH], dhv[CH];
        f32x2 dot = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
            if (i < n8) {
                dyv[c] = lds8(reinterpret_cast<const T*>(ring.at(ring.stage, 0)) + i * 8);
                hv[c] = lds8(reinterpret_cast<const T*>(ring.at(ring.stage, 1)) + i * 8);
                if (past) dhv[c] = lds8(reinterpret_cast<const T*>(ring.at(ring.stage, 2)) + i * 8);
                f32x2 d[4], n[4], w[4];
                unpack8(dyv[c], d);
                unpack8(hv[c], n);
                unpack8(wv[c], w);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    n[j] = mul2(n[j], rstd2);
                    dw[c][j] = fma2(d[j], n[j], dw[c][j]);
                    dot = fma2(mul2(d[j], w[j]), n[j], dot);
                }
            }
        }
        const float mean = __fdiv_rn(block_sum(lo2(dot) + hi2(dot), sums + flip), (float)p.H);
        const long long ahead = (long long)row + (long long)p.stages * step;
        if (threadIdx.x == 0 && ring.live && ahead < p.T) fetch(ring.stage, (int)ahead);
        ring.next();
        const f32x2 minus_mean = both(-mean);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = c * blockDim.x + threadIdx.x;
            if (i < n8) {
                f32x2 d[4], n[4], w[4];
                unpack8(dyv[c], d);
                unpack8(hv[c], n);
                unpack8(wv[c], w);
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = mul2(rstd2, fma2(mul2(n[j], rstd2), minus_mean, mul2(d[j], w[j])));
                if (past) {
                    unpack8(dhv[c], n);
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] = add2(d[j], n[j]);
                }
                store8_streaming(static_cast<T*>(p.dx) + (long long)row * p.H + i * 8, pack8<T>(d));
            }
        }
        if (p.T - row <= step) break;
        row += step;
    }
    ring.leave();
    pdl_launch_dependents();                   // the kernel that adds the shares up may be scheduled; it waits for this one's end
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i < n8) store8(p.partial + (long long)blockIdx.x * p.H + i * 8, pack8<float>(dw[c]));
    }
}

// dw[c] = sum of the blocks' shares, always in the same order.  Block: 32 columns x 32 strands of blocks.
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* partial, float* __restrict__ dw, int parts, int H) {
    __shared__ float t[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    float s = 0.0f;
    pdl_wait();
    if (c < H)
#pragma unroll 8
        for (int i = strand; i < parts; i += 32) s += partial[(long long)i * H + c];
    t[strand][threadIdx.x & 31] = s;
    __syncthreads();
    s = warp_sum(t[threadIdx.x & 31][strand]);
    const int col = blockIdx.x * 32 + strand;
    if ((threadIdx.x & 31) == 0 && col < H) dw[col] = s;
}

}  // namespace b200
