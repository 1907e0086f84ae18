// Top-k routing from the logits of one token per warp, and its gradient.
//
//   score   p_e = exp(l_e - max) / sum_i exp(l_i - max)   or   p_e = 1 / (1 + exp(-l_e))
//   key     p_e + bias_e: it chooses the experts and is not part of the weights
//   groups  n_group runs of E / n_group experts; a group counts for its best key, or the sum of its two best; only the
//           experts of the topk_group best groups can be chosen
//   weight  w_j = p_j, or p_j / (sum of the chosen p + 1e-20); times `scale`
//   gradient  with G_j = dL/dw_j * scale and S the sum: dL/dp_j = G_j, or (G_j - sum(G p) / S) / S over the chosen;
//           dl_e = p_e ([e chosen] dL/dp_e - sum over the chosen of dL/dp p), or dL/dp_e p_e (1 - p_e)
//
// An expert whose logit is -infinity or NaN is switched off: no score, never chosen.  Where fewer than top_k experts are
// left, the id is -1 and the weight 0.
//
// Which experts are chosen follows the order of the keys in 64 bits, ties to the lowest index.  Without a bias that order is
// the logits' own.  With one, or between groups, the fp32 keys decide only where they are further apart than their error
// (rt_margin); where they are not, keys in 64 bits do.  How often that is depends on the data, and equal keys count: 16384 x 256
// in groups, sigmoid: 19 us with fp32 logits of deviation 1.5 (a few tokens in a thousand), 22 us with deviation 6 (the best keys
// lie next to 1), 25 us with bf16 logits and a bias of zeros (a third of the tokens have equal keys among their best).
//
// Bound by the instructions of the choice, not by memory.  The choice has no round per expert: the best key of each lane is
// sorted across the warp; the top_k-th of them is a bound that top_k keys at least reach; the few keys that do (about a
// dozen) are collected, one to a lane, and each counts how many are before it.  16384 x 256 with bias and groups, top 8:
// 51 us with a reduction over the warp per chosen expert, 20 us like this.
#pragma once

#include "num_common.cuh"

namespace b200 {

constexpr int RT_WARPS = 4;
constexpr int RT_MAX_E = 1024;
constexpr int RT_MAX_GROUPS = 32;

struct RouteParams {
    const void* logits; long long stride;
    const void* bias; int bias_bf16;    // may be null
    int* ids;
    float* weights;
    int T, E, top_k, n_group, topk_group;
    int sigmoid, top2, renorm, vec, bias_vec;
    int gs;                             // experts per group
    int group_shift;                    // a group is 2^group_shift whole lanes; -1: lanes and groups do not match
    float scale;
};

__device__ __forceinline__ bool rt_off(float l) { return !(l > -INFINITY); }        // -infinity or NaN
constexpr float RT_BIG = 3.402823466e38f;           // +infinity counts as the largest number
__device__ __forceinline__ float rt_bias(const RouteParams& p, int e) {
    const float b = p.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[e]) : __ldg(static_cast<const float*>(p.bias) + e);
    return b > RT_BIG ? RT_BIG : b;                 // a NaN stays one
}
// larger key = larger number; 0 is below every key
__device__ __forceinline__ uint32_t rt_order(float f) {
    const uint32_t b = __float_as_uint(f);
    return b ^ (((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float rt_unorder(uint32_t o) {
    return __uint_as_float(o ^ (((int32_t)~o >> 31) | 0x80000000u));
}
// How far apart two fp32 keys must be for their order to be the exact one: `unit` times the larger of 1 and their magnitude.
// With u = 2^-24, an exponential's argument is off by three roundings (the difference, log2(e), the product) and exp2 by 4 u,
// so exp(x) by (3 |x| + 4) u of itself.
//   sigmoid   p (1 - p) (2 |l| + 4) u + 3 u p for the sum 1 + exp and the reciprocal: at most 4.5 u, as p (1 - p) |l| < 0.23;
//             two keys, and half a step of each for the bias: 11 u.  RT_UNIT_SIGMOID is 16 u
//   softmax   the sum of the exponentials adds PER - 1 + 5 roundings and the average of its terms' errors, (3 a + 4) u with
//             a = sum p |x|; the reciprocal and the product two more: p (3 |x| + 3 a + PER + 14) u, where p |x| <= 1 / e and
//             p a <= (1 - p) p ln(1023 p / (1 - p)) < 1.77.  Two keys have p + p' <= 1: (PER + 14 + 2 (3 * 1.77 + 1.11)) u, and 2 u
//             for the bias: PER + 29.  rt_unit gives PER + 32.  (1024 experts of which one dominates: 31 u are reached)
// A group's sum of two keys has the errors of both, by the larger one's magnitude however much of it cancels, and a rounding:
// two groups of two such keys stay below 2 (PER + 32) u (sigmoid: 26 u).
constexpr float RT_UNIT_SIGMOID = 16.0f / 16777216.0f;
template <int PER> __device__ __forceinline__ float rt_unit(bool sigmoid) { return sigmoid ? RT_UNIT_SIGMOID : (PER + 32) / 16777216.0f; }
__device__ __forceinline__ float rt_margin(float key, float unit) { return unit * fmaxf(1.0f, fabsf(key)); }

__device__ __forceinline__ float rt_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rt_exp(float x) { return rt_ex2(x * 1.4426950408889634f); }
__device__ __forceinline__ float rt_sigmoid(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + rt_exp(-x)));
    return r;
}

// PER consecutive values; -infinity behind E and for NaN, +0 for -0 (equal numbers, but rt_order goes by the bits).  vec:
// whole 16-byte pieces (E, the row distance and the base allow it).
template <typename T, int PER>
__device__ __forceinline__ void rt_load(const T* row, int E, int lane, bool vec, float (&l)[PER]) {
    constexpr int VL = PER < (int)(16 / sizeof(T)) ? PER : (int)(16 / sizeof(T));
    if (vec) {
#pragma unroll
        for (int j = 0; j < PER; j += VL) {
            struct alignas(sizeof(T) * VL) V { T v[VL]; } x;
            const bool in = lane * PER + j < E;
            if (in) x = *reinterpret_cast<const V*>(row + lane * PER + j);
#pragma unroll
            for (int i = 0; i < VL; ++i) l[j + i] = in ? to_f32(x.v[i]) : -INFINITY;
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) l[j] = lane * PER + j < E ? to_f32(row[lane * PER + j]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) l[j] = fminf(fmaxf(l[j] + 0.0f, -INFINITY), RT_BIG);
}

// Softmax statistics of the row: its largest logit and 1 / the sum of the exponentials (0 where every expert is off);
// e[j]: the exponentials, 0 for an expert that is off.
template <int PER>
__device__ __forceinline__ void rt_softmax(const float (&l)[PER], float (&e)[PER], float* mx, float* inv) {
    float m = l[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) m = fmaxf(m, l[j]);
    m = warp_max(m);
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        e[j] = rt_exp(l[j] - m);
        s += e[j];
    }
    s = warp_sum(s);
    *mx = m;
    *inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
}
// the score of one expert that is not off, for its weight
__device__ __forceinline__ float rt_score(float l, bool sigmoid, float mx, float inv) {
    return sigmoid ? __fdiv_rn(1.0f, 1.0f + expf(-l)) : expf(fminf(l, RT_BIG) - mx) * inv;
}

// ---- 64 bits, for the tokens whose fp32 keys are too close.  The whole warp takes part in each.
// Softmax: the row's largest logit and the sum of the exponentials.
template <typename T>
__device__ __forceinline__ void rt_softmax64(const RouteParams& p, const T* row, int lane, double* mx, double* sum) {
    float m = -INFINITY;
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, to_f32(row[e]));
    m = fminf(warp_max(m), RT_BIG);
    double s = 0.0;
    for (int e = lane; e < p.E; e += 32) {
        const float l = to_f32(row[e]);
        if (!rt_off(l)) s += exp((double)fminf(l, RT_BIG) - (double)m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    *mx = m;
    *sum = s;
}
__device__ __forceinline__ double rt_key64_of(const RouteParams& p, float l, int e, double mx, double sum) {
    const double k = p.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)fminf(l, RT_BIG) - mx) / sum;
    return p.bias ? k + (double)rt_bias(p, e) : k;
}
// The key of expert `id` (-1: none).
template <typename T>
__device__ __noinline__ double rt_key64(const RouteParams& p, const T* row, int id, int lane) {
    double mx = 0.0, sum = 1.0;
    if (!p.sigmoid) rt_softmax64<T>(p, row, lane, &mx, &sum);
    return id >= 0 ? rt_key64_of(p, to_f32(row[id]), id, mx, sum) : -INFINITY;
}
// The keys of all experts, -infinity for one that is off.
template <typename T>
__device__ __noinline__ void rt_keys64(const RouteParams& p, const T* row, double* key, int lane) {
    double mx = 0.0, sum = 1.0;
    if (!p.sigmoid) rt_softmax64<T>(p, row, lane, &mx, &sum);
    for (int e = lane; e < p.E; e += 32) {
        const float l = to_f32(row[e]);
        const double k = rt_off(l) ? (double)-INFINITY : rt_key64_of(p, l, e, mx, sum);
        key[e] = k > (double)-INFINITY ? k : (double)-INFINITY;          // a NaN in the bias
    }
    __syncwarp();
}
// Whether group `lane` is among the topk_group best.
template <typename T>
__device__ __noinline__ bool rt_groups64(const RouteParams& p, const T* row, double* key, int lane) {
    rt_keys64<T>(p, row, key, lane);
    double a = -INFINITY, b = -INFINITY;
    if (lane < p.n_group)
        for (int i = 0; i < p.gs; ++i) {
            const double k = key[lane * p.gs + i];
            b = fmax(b, fmin(a, k));
            a = fmax(a, k);
        }
    const double g = p.top2 && b > (double)-INFINITY ? a + b : a;
    int before = 0;
    for (int i = 0; i < p.n_group; ++i) {
        const double o = __shfl_sync(0xffffffffu, g, i);
        before += o > g || (o == g && i < lane);
    }
    __syncwarp();
    return lane < p.n_group && before < p.topk_group;
}
// The choice one expert after the other from keys in shared memory -> the id of choice `lane` (-1: none).
__device__ __noinline__ int rt_choose64(int E, int top_k, double* key, int lane) {
    int mine = -1;
    for (int k = 0; k < top_k; ++k) {
        double best = -INFINITY;
        int at = -1;
        for (int e = lane; e < E; e += 32)
            if (key[e] > best) { best = key[e]; at = e; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa >= 0 && (at < 0 || oa < at))) { best = ob; at = oa; }
        }
        if (at < 0) break;
        if (lane == k) mine = at;
        if (lane == (at & 31)) key[at] = -INFINITY;
        __syncwarp();
    }
    return mine;
}

constexpr uint32_t RT_LEAST = 0x00800000u;          // rt_order of the lowest number; -infinity is one less

// One warp per token; lane l holds experts l * PER ... l * PER + PER - 1.
template <typename T, int PER>
__global__ void __launch_bounds__(RT_WARPS * 32) route_kernel(const RouteParams p) {
    extern __shared__ double rt_smem[];              // per warp: E 64-bit keys (where keys are scores)
    __shared__ unsigned long long cands[RT_WARPS][2][32];          // key << 32 | ~expert: the larger one comes first
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * RT_WARPS + warp;
    if (t >= p.T) return;
    double* key64 = rt_smem + warp * p.E;
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    float l[PER], k[PER];
    rt_load<T, PER>(row, p.E, lane, p.vec, l);
    float mx = 0.0f, inv = 0.0f;
    if (!p.sigmoid) rt_softmax(l, k, &mx, &inv);
    const bool scored = p.bias != nullptr || p.n_group > 1;
    const float unit = rt_unit<PER>(p.sigmoid);
    if (scored) {
#pragma unroll
        for (int j = 0; j < PER; ++j) k[j] = p.sigmoid ? rt_sigmoid(l[j]) : k[j] * inv;
        if (p.bias) {
            float b[PER];
            if (p.bias_bf16) rt_load<__nv_bfloat16, PER>(static_cast<const __nv_bfloat16*>(p.bias), p.E, lane, p.bias_vec, b);
            else rt_load<float, PER>(static_cast<const float*>(p.bias), p.E, lane, p.bias_vec, b);
#pragma unroll
            for (int j = 0; j < PER; ++j) k[j] += b[j];
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) k[j] = l[j] == -INFINITY ? -INFINITY : k[j];
    }
    uint32_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = rt_order(p.bias ? k[j] : l[j]);
    if (p.n_group > 1) {
        const bool even = p.group_shift >= 0;
        float a = -INFINITY, b = -INFINITY;            // the two best keys of a lane, then of a group
        if (even) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                b = fmaxf(b, fminf(a, k[j]));
                a = fmaxf(a, k[j]);
            }
            for (int o = 1; o < 1 << p.group_shift; o <<= 1) {
                const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
                b = fmaxf(fminf(a, oa), fmaxf(b, ob));
                a = fmaxf(a, oa);
            }
        } else {
            float* skey = reinterpret_cast<float*>(key64);
#pragma unroll
            for (int j = 0; j < PER; ++j) if (lane * PER + j < p.E) skey[lane * PER + j] = k[j];
            __syncwarp();
            if (lane < p.n_group)
                for (int i = 0; i < p.gs; ++i) {
                    const float v = skey[lane * p.gs + i];
                    b = fmaxf(b, fminf(a, v));
                    a = fmaxf(a, v);
                }
            __syncwarp();
        }
        const int shift = even ? p.group_shift : 0, g_of = lane >> shift;          // lane g << shift has group g's score
        const bool pair = p.top2 && b > -INFINITY;
        // a sum past the range is held at its end, next to the others there, and above a group without experts
        const float g = pair ? fminf(fmaxf(a + b, -RT_BIG), RT_BIG) : a,
                    eps = 2.0f * rt_margin(fmaxf(fabsf(a), pair ? fabsf(b) : 0.0f), unit);
        int before = 0, near = 0;
        for (int i = 0; i < p.n_group; ++i) {
            const float o = __shfl_sync(0xffffffffu, g, i << shift);
            before += o > g || (o == g && i < g_of);
            near += fabsf(o - g) <= eps;              // itself, and groups whose order needs 64 bits
        }
        bool kept = g_of < p.n_group && before < p.topk_group;
        const bool real = g_of < p.n_group && g > -INFINITY;
        unsigned keep = __ballot_sync(0xffffffffu, kept);
        if (__any_sync(0xffffffffu, real && near > 1)) {           // it matters where one is kept and the other is not
            bool close = false;
            for (int i = 0; i < p.n_group; ++i) {
                const float o = __shfl_sync(0xffffffffu, g, i << shift);
                close |= real && fabsf(o - g) <= eps && kept != (bool)((keep >> (i << shift)) & 1u);
            }
            if (__any_sync(0xffffffffu, close)) {
                const unsigned groups = __ballot_sync(0xffffffffu, rt_groups64<T>(p, row, key64, lane));
                kept = (groups >> g_of) & 1u;
                keep = __ballot_sync(0xffffffffu, kept);
            }
        }
        if (even) {
#pragma unroll
            for (int j = 0; j < PER; ++j) key[j] = kept ? key[j] : 0u;
        } else {
            int g_at = lane * PER / p.gs, left = (g_at + 1) * p.gs - lane * PER;       // of that group from this expert on
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (left == 0) { ++g_at; left = p.gs; }
                --left;
                if (!((keep >> (g_at & 31)) & 1u)) key[j] = 0u;
            }
        }
    }
    int mine = -1;
    // with a bias the best key left out is looked at too
    const int wanted = p.bias ? p.top_k + 1 : p.top_k;
    uint32_t bound = key[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) bound = max(bound, key[j]);
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, bound, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);
            bound = larger ? max(bound, other) : min(bound, other);
        }
    bound = __shfl_sync(0xffffffffu, bound, min(wanted, 32) - 1);
    if (p.bias && bound >= RT_LEAST) {              // whatever 64 bits may put among the chosen is collected too
        const float v = rt_unorder(bound);
        bound = rt_order(v - rt_margin(v, unit));
    }
    bound = max(bound, RT_LEAST);
    int count = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) count += key[j] >= bound;
    int at = count;                                  // where this lane's candidates begin
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += v;
    }
    const int total = __shfl_sync(0xffffffffu, at, 31);
    at -= count;
    if (total <= 32 && wanted <= 32) {
        unsigned long long* c = cands[warp][0];
        unsigned long long* sorted = cands[warp][1];
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (key[j] >= bound) c[at++] = (unsigned long long)key[j] << 32 | (uint32_t)~(lane * PER + j);
        __syncwarp();
        const unsigned long long me = lane < total ? c[lane] : 0ull;
        int rank = 0;
        for (int i = 0; i < total; ++i) rank += c[i] > me;
        if (lane < total) sorted[rank] = me;
        __syncwarp();
        const unsigned long long s = lane < total ? sorted[lane] : 0ull;
        mine = lane < total ? (int)~(uint32_t)s : -1;
        if (p.bias) {
            const float v = rt_unorder((uint32_t)(s >> 32));
            const float next = __shfl_down_sync(0xffffffffu, v, 1);
            if (__any_sync(0xffffffffu, lane < p.top_k && lane + 1 < total && v - next <= rt_margin(v, unit))) {
                const double exact = rt_key64<T>(p, row, mine, lane);
                rank = 0;
                for (int i = 0; i < total; ++i) {
                    const double o = __shfl_sync(0xffffffffu, exact, i);
                    const int oe = __shfl_sync(0xffffffffu, mine, i);
                    rank += o > exact || (o == exact && oe < mine);
                }
                __syncwarp();
                if (lane < total) c[rank] = s;
                __syncwarp();
                if (lane < total) mine = (int)~(uint32_t)c[lane];
            }
        }
    } else {
        // many equal keys: one after the other
        bool close = false;
        float last = INFINITY;
        unsigned allowed = 0;                        // of this lane's experts
#pragma unroll
        for (int j = 0; j < PER; ++j) allowed |= (unsigned)(key[j] >= RT_LEAST) << j;
        for (int r = 0; r < wanted; ++r) {
            uint32_t best = key[0];
            int a = 0;
#pragma unroll
            for (int j = 1; j < PER; ++j) if (key[j] > best) { best = key[j]; a = j; }
            const uint32_t m = __reduce_max_sync(0xffffffffu, best);
            if (m < RT_LEAST) break;
            const int winner = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
            const int e = __shfl_sync(0xffffffffu, lane * PER + a, winner);
            if (lane == r) mine = e;
            if (lane == winner) {
#pragma unroll
                for (int j = 0; j < PER; ++j) if (j == a) key[j] = 0u;
            }
            if (p.bias) {
                const float v = rt_unorder(m);
                close |= last - v <= rt_margin(v, unit);
                last = v;
            }
        }
        if (close) {                                 // the same in all lanes
            rt_keys64<T>(p, row, key64, lane);
            for (int j = 0; j < PER; ++j)
                if (lane * PER + j < p.E && !((allowed >> j) & 1u)) key64[lane * PER + j] = -INFINITY;
            __syncwarp();
            mine = rt_choose64(p.E, p.top_k, key64, lane);
        }
    }
    if (lane >= p.top_k) mine = -1;
    const float s = mine >= 0 ? rt_score(to_f32(row[mine]), p.sigmoid, mx, inv) : 0.0f;
    const float total_s = warp_sum(s) + 1e-20f;
    if (lane < p.top_k) {
        p.ids[(long long)t * p.top_k + lane] = mine;
        p.weights[(long long)t * p.top_k + lane] = (p.renorm ? __fdiv_rn(s, total_s) : s) * p.scale;
    }
}

struct RouteGradParams {
    const float* grad;                  // [T, top_k]
    const void* logits; long long stride;
    const int* ids;
    void* out;                          // [T, E], dense, the logits' type
    int T, E, top_k, sigmoid, renorm, vec;
    float scale;
};

// One warp per token.  A row is -p_e * sum(G p) of the chosen (softmax) or 0 everywhere but at the chosen experts, which are
// written over it.  There the formulas at the head of this file subtract numbers that are nearly equal once one score
// dominates; from 1 = sum of all p the same is, without a difference but those of the G,
//   renormalised  dL/dp_j = (sum over the chosen of (G_j - G_k) p_k + 1e-20 G_j) / S^2
//   softmax       dl_j = p_j (sum over the chosen of (G_j - G_k) p_k + G_j * the sum of the other experts' p)
// Bound by memory's latency.
template <typename T, int PER>
__global__ void __launch_bounds__(RT_WARPS * 32) route_grad_kernel(const RouteGradParams p) {
    __shared__ unsigned marks[RT_WARPS][32];   // a bit for each expert that is chosen
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * RT_WARPS + warp;
    if (t >= p.T) return;
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    int id = -1;
    float g = 0.0f, s = 0.0f, li = -INFINITY;
    if (lane < p.top_k) {
        id = __ldg(p.ids + (long long)t * p.top_k + lane);
        g = __ldg(p.grad + (long long)t * p.top_k + lane) * p.scale;
    }
    float o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = 0.0f;
    float mx = 0.0f, inv = 0.0f;
    if (!p.sigmoid) {
        float l[PER];
        rt_load<T, PER>(row, p.E, lane, p.vec, l);
        if (id >= 0 && id < p.E) li = to_f32(row[id]);
        rt_softmax(l, o, &mx, &inv);
    } else if (id >= 0 && id < p.E) li = to_f32(row[id]);
    if (rt_off(li)) {
        id = -1;
        g = 0.0f;
    } else s = rt_score(li, p.sigmoid, mx, inv);
    marks[warp][lane] = 0u;
    __syncwarp();
    if (id >= 0) atomicOr(&marks[warp][id / PER], 1u << (id % PER));
    // dL/dp of each choice.  (Products with 1 / S: a division of numbers near 1e-20 took 15 us of 16384 tokens' 26.)
    float minus = 0.0f;
    if (p.renorm) {
        const float total = warp_sum(s) + 1e-20f, r = __frcp_rn(total), dot = warp_sum(g * s);
        float d = g * 1e-20f;
        for (int k = 0; k < p.top_k; ++k) d = fmaf(g - __shfl_sync(0xffffffffu, g, k), __shfl_sync(0xffffffffu, s, k), d);
        g = id >= 0 ? d * r * r : 0.0f;
        minus = -(dot * r) * (1e-20f * r);                   // the sum of g s: all but the 1e-20 cancels
    } else if (!p.sigmoid) minus = -warp_sum(g * s);
    __syncwarp();
    const unsigned chosen = marks[warp][lane];               // of this lane's experts
    bool first = true;
    if ((int)__reduce_add_sync(0xffffffffu, __popc(chosen)) != __popc(__ballot_sync(0xffffffffu, id >= 0))) {
        // of an expert that a token names twice: the sum of both, which both lanes add up in the same order
        const unsigned same = __match_any_sync(0xffffffffu, id);
        float sum = 0.0f;
        for (int k = 0; k < p.top_k; ++k) {
            const float og = __shfl_sync(0xffffffffu, g, k);
            if ((same >> k) & 1u) sum += og;
        }
        g = sum;
        first = __ffs(same) - 1 == lane;
    }
    float mine;                                // the gradient at expert id
    if (p.sigmoid) mine = g * s * __fdiv_rn(1.0f, 1.0f + expf(li));          // 1 - s, which loses its bits as s nears 1
    else if (p.renorm) mine = s * (g + minus);
    else {
        const float once = first ? s : 0.0f;
        float d = 0.0f, rest = 0.0f;
        for (int k = 0; k < p.top_k; ++k) d = fmaf(g - __shfl_sync(0xffffffffu, g, k), __shfl_sync(0xffffffffu, once, k), d);
#pragma unroll
        for (int j = 0; j < PER; ++j) rest += (chosen >> j) & 1u ? 0.0f : o[j];
        mine = s * fmaf(g, warp_sum(rest) * inv, d);
    }
    if (!p.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] *= minus * inv;
    }
    T* out = static_cast<T*>(p.out) + (long long)t * p.E;
    if (p.vec) {
        constexpr int VL = PER < (int)(16 / sizeof(T)) ? PER : (int)(16 / sizeof(T));
#pragma unroll
        for (int j = 0; j < PER; j += VL) {
            struct alignas(sizeof(T) * VL) V { T v[VL]; } x;
#pragma unroll
            for (int i = 0; i < VL; ++i) x.v[i] = from_f32<T>(o[j + i]);
            if (lane * PER + j < p.E) *reinterpret_cast<V*>(out + lane * PER + j) = x;
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) if (lane * PER + j < p.E) out[lane * PER + j] = from_f32<T>(o[j]);
    }
    __syncwarp();
    if (id >= 0) out[id] = from_f32<T>(mine);
}

}  // namespace b200
