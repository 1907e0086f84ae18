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
// Bound by memory: a thread holds the 16 columns of several rows at a time, so that enough loads are under way.
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
__device__ __forceinline__ uint32_t pack8_e2m1(const f32x2 (&v)[4]) {
    uint16_t h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        asm("{\n\t.reg .b8 a, b;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "mov.b16 %0, {a, b};\n\t}"
            : "=h"(h[i]) : "f"(lo2(v[2 * i])), "f"(hi2(v[2 * i])), "f"(lo2(v[2 * i + 1])), "f"(hi2(v[2 * i + 1])));
    uint32_t r;
    asm("mov.b32 %0, {%1, %2};" : "=r"(r) : "h"(h[0]), "h"(h[1]));
    return r;
}

// The larger magnitudes of two pairs of 16-bit values; a NaN stays one.
template <typename T> __device__ __forceinline__ uint32_t amax2_nan(uint32_t m, uint32_t u);
template <> __device__ __forceinline__ uint32_t amax2_nan<__nv_bfloat16>(uint32_t m, uint32_t u) {
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tabs.bf16x2 t, %2;\n\tmax.NaN.bf16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(m), "r"(u));
    return r;
}
template <> __device__ __forceinline__ uint32_t amax2_nan<__half>(uint32_t m, uint32_t u) {
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tabs.f16x2 t, %2;\n\tmax.NaN.f16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(m), "r"(u));
    return r;
}
// The largest magnitude of 16 values.
template <typename T> __device__ __forceinline__ float largest16(const Raw8<T>& a, const Raw8<T>& b) {
    uint32_t m = 0;
    const uint32_t u[8] = {a.w[0].x, a.w[0].y, a.w[0].z, a.w[0].w, b.w[0].x, b.w[0].y, b.w[0].z, b.w[0].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) m = amax2_nan<T>(m, u[i]);
    const f32x2 f = Fmt<T>::up(m);
    return amax_nan(lo2(f), hi2(f));
}
template <> __device__ __forceinline__ float largest16<float>(const Raw8<float>& a, const Raw8<float>& b) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint4 w = i < 2 ? a.w[i & 1] : b.w[i & 1];
        m = max(max(m, w.x & 0x7FFFFFFFu), max(w.y & 0x7FFFFFFFu, max(w.z & 0x7FFFFFFFu, w.w & 0x7FFFFFFFu)));
    }
    return __uint_as_float(m);
}

// x / (1 + exp(-x)) with the hardware's exp2 and reciprocal: off by at most (1.25 |x| + 8) 2^-24 of the value (exp2's argument
// by the product's rounding and the constant's, 1.25 |x| 2^-24 of exp; exp2 4, the sum 1, the reciprocal 2, the product 1 times
// 2^-24): 2e-6 at |x| = 20, a ten-thousandth of a 4-bit step.  From x = -87.4 down, where the value is below 2^-119, the
// reciprocal is flushed and the result 0.
__device__ __forceinline__ float silu_quick(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * r;
}

// One nvfp4 block by CUDA's division: its codes, and its scale byte as the result.  For factors at the ends of the range and
// for values that overflow against the largest scale; a block that is not finite keeps the zeros it has.  Behind the loop over
// the rows: 68 such divisions inside it took registers from every block (16384 x 7168: 58 us instead of 54).
template <typename T, bool SILU>
__device__ __forceinline__ uint8_t divided_block(const T* gate, const T* up, float g, uint8_t* q) {
    f32x2 v[2][4];
    float amax = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        unpack8(load8(gate + 8 * h), v[h]);
        if (SILU) {
            f32x2 w[4];
            unpack8(load8(up + 8 * h), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[h][j] = mul2(pack_f32x2(silu_quick(lo2(v[h][j])), silu_quick(hi2(v[h][j]))), w[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = amax_nan(amax_nan(amax, lo2(v[h][j])), hi2(v[h][j]));
    }
    if (!(amax < INFINITY)) return 0x7F;
    const __nv_fp8_storage_t byte = __nv_cvt_float_to_fp8(fminf(__fdiv_rn(amax, __fmul_rn(6.0f, g)), 448.0f), __NV_SATFINITE, __NV_E4M3);
    const float unit = __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3))), g);
    if (unit > 0.0f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j >> 2][j & 3] = pack_f32x2(__fdiv_rn(lo2(v[j >> 2][j & 3]), unit), __fdiv_rn(hi2(v[j >> 2][j & 3]), unit));
        *reinterpret_cast<uint2*>(q) = make_uint2(pack8_e2m1(v[0]), pack8_e2m1(v[1]));
    }
    return byte;
}

constexpr int FP4_QUANT_THREADS = 256, FP4_QUANT_ROWS = 64;

// NV: nvfp4, else mxfp4.  SILU: x holds gate and up, K columns each.  BY_ROW: scales row after row, for copy_fp4_rows_kernel.
// Block: 64 rows x 256 columns.  A thread takes 16 columns of a row at a time (a block of nvfp4, half a block of mxfp4) and
// four such rows in all: of 16-bit inputs all four are loaded before the first is used, of the others two at a time.
// Blocks per SM as measured (16384 x 7168 nvfp4: 3, 4, 5 blocks 59, 55, 53 us; mxfp4: 4, 5, 6 blocks 48, 46, 61 us; SiLU*mul of
// 16384 x 2048: 2, 3, 4 blocks 42, 31, 31 us).  mxfp4 runs at memory's speed (45 us, 6.5 TB/s); nvfp4 has a division more per
// value and is bound by its instructions (53 us, 5.7 TB/s).  What it divides by has one value per scale byte: the block tables
// them with their reciprocals.
template <typename T, bool NV, bool SILU, bool BY_ROW>
__global__ void __launch_bounds__(FP4_QUANT_THREADS, sizeof(T) == 2 ? (SILU ? 3 : 5) : 2) quant_fp4_kernel(const Fp4QuantParams p) {
    constexpr int WORDS = NV ? 4 : 2;           // scale tiles of 256 columns
    constexpr int STEP = FP4_QUANT_THREADS / 16, ROWS = FP4_QUANT_ROWS / STEP, BATCH = sizeof(T) == 2 && !SILU ? ROWS : ROWS / 2;
    __shared__ uint32_t tile[WORDS][FP4_QUANT_ROWS];
    __shared__ float2 units[NV ? 128 : 1];      // of a scale byte: minus s g, and 1 / (s g), 0 for the scale zero
    const int group = blockIdx.y, row_pieces = ((p.rows + 127) >> 7) * (128 / FP4_QUANT_ROWS);
    const int rb = blockIdx.x / p.k_blocks, kb = blockIdx.x - rb * p.k_blocks;
    const int r0 = rb * FP4_QUANT_ROWS, i0 = threadIdx.x >> 4;
    const int seg = threadIdx.x & 15, col = kb * 256 + seg * 16;
    const float g = p.factor ? __ldg(p.factor + group * p.factor_stride) : 1.0f;
    const float g6 = __fmul_rn(6.0f, g), r6 = __frcp_rn(g6);
    const bool near = g > 1e-27f && g < 1e26f;  // div_by can divide by 6 g and by every scale but zero
    const T* xg = static_cast<const T*>(p.x) + (long long)group * p.src_rows * p.x_stride + col;
    const int gate = SILU && !p.gate_first ? p.K : 0, up = p.gate_first ? p.K : 0;
    int src[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const int r = r0 + i0 + k * STEP;
        src[k] = r < p.rows && col < p.K ? (p.src ? __ldg(p.src + r) : r) : -1;
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        if (p.src && src[k] >= 0) src[k] = src[k] / p.top_k;
        if (src[k] >= p.src_rows) src[k] = -1;
    }
    unsigned again = 0;                         // rows whose block is left to divided_block
#pragma unroll
    for (int b = 0; b < ROWS; b += BATCH) {
        Raw8<T> x[BATCH][2], u[SILU ? BATCH : 1][2];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            if (src[b + k] < 0) continue;
            const T* row = xg + src[b + k] * p.x_stride;
            x[k][0] = load8(row + gate);
            x[k][1] = load8(row + gate + 8);
            if (SILU) {
                u[k][0] = load8(row + up);
                u[k][1] = load8(row + up + 8);
            }
        }
        if (NV && b == 0) {                     // while the rows are on their way
            if (threadIdx.x < 128) {
                const float unit = __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)threadIdx.x, __NV_E4M3))), g);
                units[threadIdx.x] = make_float2(-unit, unit > 0.0f ? __frcp_rn(unit) : 0.0f);
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + (b + k) * STEP;
            const bool live = src[b + k] >= 0;             // the same for all threads of a scale block
            f32x2 v[2][4];
            float amax = largest16(x[k][0], x[k][1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                unpack8(x[k][h], v[h]);
                if (SILU) {
                    f32x2 w[4];
                    unpack8(u[k][h], w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[h][j] = mul2(pack_f32x2(silu_quick(lo2(v[h][j])), silu_quick(hi2(v[h][j]))), w[j]);
                }
            }
            if (SILU) {
                amax = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = amax_nan(amax_nan(amax, lo2(v[j >> 2][j & 3])), hi2(v[j >> 2][j & 3]));
            }
            if (!NV) amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            uint32_t byte = 0;
            if (live) {
                uint2 codes;
                if (NV) {
                    const float q = __fmul_rn(amax, r6), t = __fmaf_rn(__fmaf_rn(-g6, q, amax), r6, q);       // amax / (6 g)
                    const bool fit = near && t < 1e30f;     // false for a NaN too
                    if (!fit) again |= 1u << (b + k);
                    byte = fit ? __nv_cvt_float_to_fp8(fminf(t, 448.0f), __NV_SATFINITE, __NV_E4M3) : 0x7Fu;
                    const float2 of = units[byte];
                    const f32x2 minus = both(of.x), r = both(of.y);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j >> 2][j & 3] = div_by(v[j >> 2][j & 3], minus, r);
                    codes = make_uint2(pack8_e2m1(v[0]), pack8_e2m1(v[1]));
                    if (!fit) codes = make_uint2(0u, 0u);
                } else {
                    const bool finite = amax < INFINITY;
                    byte = finite ? (uint32_t)max((int)(__float_as_uint(amax) >> 23) - 2, 0) : 0xFFu;
                    const f32x2 inv = both(__uint_as_float((254u - byte) << 23));                 // 2^(127 - byte), exact
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j >> 2][j & 3] = finite ? mul2(v[j >> 2][j & 3], inv) : 0;
                    codes = make_uint2(pack8_e2m1(v[0]), pack8_e2m1(v[1]));
                }
                *reinterpret_cast<uint2*>(p.q + ((long long)group * p.rows + r0 + i) * (p.K >> 1) + (col >> 1)) = codes;
            }
            const int blk = NV ? seg : seg >> 1;            // block of these 256 columns
            if (NV || !(seg & 1)) reinterpret_cast<uint8_t*>(&tile[blk >> 2][i])[blk & 3] = (uint8_t)byte;
        }
    }
    for (; again; again &= again - 1) {
        const int i = i0 + (__ffs(again) - 1) * STEP, r = r0 + i;
        const T* row = xg + (p.src ? __ldg(p.src + r) / p.top_k : r) * p.x_stride;
        reinterpret_cast<uint8_t*>(&tile[seg >> 2][i])[seg & 3] =
            divided_block<T, SILU>(row + gate, row + up, g, p.q + ((long long)group * p.rows + r) * (p.K >> 1) + (col >> 1));
    }
    __syncthreads();
    if (BY_ROW) {
        const int i = threadIdx.x;
        if (i < FP4_QUANT_ROWS && r0 + i < p.rows) {
            uint32_t* to = reinterpret_cast<uint32_t*>(p.sf) + ((long long)(r0 + i) * p.k_blocks + kb) * WORDS;
            if (NV) *reinterpret_cast<uint4*>(to) = make_uint4(tile[0][i], tile[1][i], tile[WORDS - 2][i], tile[WORDS - 1][i]);
            else *reinterpret_cast<uint2*>(to) = make_uint2(tile[0][i], tile[1][i]);
        }
        return;
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(p.sf) + (((long long)group * (row_pieces / (128 / FP4_QUANT_ROWS)) + (r0 >> 7)) * p.k_blocks + kb) * (WORDS * 128);
    for (int w = threadIdx.x; w < WORDS * FP4_QUANT_ROWS; w += FP4_QUANT_THREADS) {
        // neighbouring threads: the words of rows i and i + 32 lie side by side
        const int t = w / FP4_QUANT_ROWS, i = ((w & 1) << 5) + ((w % FP4_QUANT_ROWS) >> 1), r = r0 + i;
        // rows that are left alone keep their scales; those behind the last one are zero
        if (p.src == nullptr || r >= p.rows || __ldg(p.src + r) >= 0) out[t * 128 + (r & 31) * 4 + ((r >> 5) & 3)] = tile[t][i];
    }
}

// Row r of (q, sf) <- row src[r] / top_k of (q0, sf0), x quantised once; the rows left alone are quant_fp4_kernel's.
// Where every row of x goes to several rows, its quantisation (53 us for 16384 x 7168 nvfp4, bound by instructions) and this
// copy (bound by the L2 cache: it reads and writes 132 MB each in 36 us for 32768 rows) beat a quantisation of each row:
// 16384 x 7168 in 2 rows each 113 -> 89 us, 4096 x 7168 in 8 rows each 108 -> 46 us.  FP4_COPY_FROM says from where on.
// The rule counts rows, of which many may be padding: a plan of 16384 tokens with 8 of 256 experts each has 131072 rows and more
// however few experts are local.  Copying is the faster way there too, because the other kernel pays for every block of rows, live
// or not: 256, 32 and 4 local experts 188, 97 and 85 us against 475, 190 and 151.
// Block: 64 rows x 1024 columns; a warp copies the 512 bytes of a row's codes and has eight rows under way.
struct Fp4CopyParams {
    const uint8_t* q0; const uint32_t* sf0;     // sf0: row after row
    const int* src; int top_k;
    uint8_t* q; uint32_t* sf;
    int rows, src_rows, K, k_blocks, pieces;
};
constexpr int FP4_COPY_COLS = 1024;
// Values from which a second kernel costs less than it saves (twice the rows of x or more; 3.7 million: 5 us without and 6 us
// with it, 8.4 million: 6.5 and 6.0 us, 14.7 million: 9.5 and 6.8 us).  With as many rows as x has it loses a sixth.
constexpr long long FP4_COPY_FROM = 1ll << 23;
template <bool NV>
__global__ void __launch_bounds__(FP4_QUANT_THREADS) copy_fp4_rows_kernel(const Fp4CopyParams p) {
    constexpr int WARPS = FP4_QUANT_THREADS / 32, EACH = FP4_QUANT_ROWS / WARPS, WORDS = NV ? 4 : 2;
    __shared__ int from[FP4_QUANT_ROWS];        // -1: leave the row alone; -2: zero scales
    const int rb = blockIdx.x / p.pieces, piece = blockIdx.x - rb * p.pieces, r0 = rb * FP4_QUANT_ROWS;
    if (threadIdx.x < FP4_QUANT_ROWS) {
        const int r = r0 + threadIdx.x, pair = r < p.rows ? __ldg(p.src + r) : 0;
        const int f = r < p.rows ? (pair >= 0 ? pair / p.top_k : -1) : -2;
        from[threadIdx.x] = f < p.src_rows ? f : -2;
    }
    __syncthreads();
    pdl_wait();
    const int col = piece * (FP4_COPY_COLS / 2) + (threadIdx.x & 31) * 16, half = p.K >> 1;
    uint4 c[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int f = from[(threadIdx.x >> 5) + j * WARPS];
        if (f >= 0 && col < half) c[j] = *reinterpret_cast<const uint4*>(p.q0 + (long long)f * half + col);
    }
    // a thread takes a row's scales of 256 columns; neighbouring threads: rows i and i + 32, whose words lie side by side
    static_assert(FP4_COPY_COLS / 256 * FP4_QUANT_ROWS == FP4_QUANT_THREADS);
    const int kb = piece * (FP4_COPY_COLS / 256) + threadIdx.x / FP4_QUANT_ROWS;
    const int i = ((threadIdx.x & 1) << 5) + ((threadIdx.x % FP4_QUANT_ROWS) >> 1), f = from[i], r = r0 + i;
    if (f != -1 && kb < p.k_blocks) {
        uint32_t w[WORDS] = {};
        if (f >= 0) {
            const uint32_t* at = p.sf0 + ((long long)f * p.k_blocks + kb) * WORDS;
            if (NV) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(at);
            else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(at);
        }
        uint32_t* out = p.sf + ((long long)(r >> 7) * p.k_blocks + kb) * (WORDS * 128) + (r & 31) * 4 + ((r >> 5) & 3);
#pragma unroll
        for (int t = 0; t < WORDS; ++t) out[t * 128] = w[t];
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int row = (threadIdx.x >> 5) + j * WARPS;
        if (from[row] >= 0 && col < half) __stcs(reinterpret_cast<uint4*>(p.q + (long long)(r0 + row) * half + col), c[j]);
    }
}

// Packed codes -> e4m3 values, 8 bytes to 16; a thread loads four of them before it stores the first.
constexpr int FP4_UNPACK_THREADS = 256, FP4_UNPACK_EACH = 4;
__global__ void __launch_bounds__(FP4_UNPACK_THREADS) unpack_fp4_kernel(const uint2* __restrict__ q, uint4* __restrict__ out, long long n) {
    // magnitudes 0 .5 1 1.5 | 2 3 4 6 as e4m3 bytes; a code's low three bits pick one, its fourth is the sign
    auto four = [](uint32_t c) {
        const uint32_t mag = __byte_perm(0x3C383000u, 0x4C484440u, c & 0x7777u);
        const uint32_t sign = ((c & 0x8u) << 4) | ((c & 0x80u) << 8) | ((c & 0x800u) << 12) | ((c & 0x8000u) << 16);
        return mag | sign;
    };
    const long long i0 = (long long)blockIdx.x * (FP4_UNPACK_THREADS * FP4_UNPACK_EACH) + threadIdx.x;
    uint2 w[FP4_UNPACK_EACH];
#pragma unroll
    for (int k = 0; k < FP4_UNPACK_EACH; ++k)
        if (i0 + k * FP4_UNPACK_THREADS < n) w[k] = __ldcs(q + i0 + k * FP4_UNPACK_THREADS);
#pragma unroll
    for (int k = 0; k < FP4_UNPACK_EACH; ++k)
        if (i0 + k * FP4_UNPACK_THREADS < n)
            __stcs(out + i0 + k * FP4_UNPACK_THREADS, make_uint4(four(w[k].x & 0xFFFFu), four(w[k].x >> 16), four(w[k].y & 0xFFFFu), four(w[k].y >> 16)));
}

}  // namespace b200
