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
// Which experts are chosen follows the exact order of the keys, ties to the lowest index.  Without a bias that order is
// the logits' own.  With one, or between groups, the fp32 keys decide only where they are further apart than their error;
// a token in which two compared keys are closer (a few in a thousand) is chosen again from keys in 64 bits.
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
    int sigmoid, top2, renorm, vec;
    float scale;
};

__device__ __forceinline__ bool rt_off(float l) { return !(l > -INFINITY); }        // -infinity or NaN
__device__ __forceinline__ float rt_bias(const RouteParams& p, int e) {
    return p.bias_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[e]) : __ldg(static_cast<const float*>(p.bias) + e);
}
// larger key = larger number; 0 is below every key
__device__ __forceinline__ uint32_t rt_order(float f) {
    const uint32_t b = __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rt_unorder(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
// What two keys of this size may be off together: exp, the division and the additions leave each score (at most 1)
// within 1e-6, the bias adds half a step of the key.
__device__ __forceinline__ bool rt_close(float a, float b) { return fabsf(a - b) <= 4e-6f * fmaxf(1.0f, fabsf(a)); }

// The E logits of a token in the warp's registers: lane l holds experts l * PER ... l * PER + PER - 1; -infinity where
// there is none.  vec: whole 16-byte pieces (E, the row distance and the base allow it).
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
    for (int j = 0; j < PER; ++j) if (rt_off(l[j])) l[j] = -INFINITY;
}

// Softmax statistics of the row: largest finite logit and 1 / sum of the exponentials (0 where every expert is off).
template <int PER>
__device__ __forceinline__ void rt_softmax(float (&l)[PER], float* mx, float* inv) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) { l[j] = fminf(l[j], 3.402823466e38f); m = fmaxf(m, l[j]); }
    m = warp_max(m);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) s += l[j] == -INFINITY ? 0.0f : expf(l[j] - m);
    s = warp_sum(s);
    *mx = m;
    *inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
}
__device__ __forceinline__ float rt_score(float l, bool sigmoid, float mx, float inv) {
    if (l == -INFINITY) return 0.0f;
    return sigmoid ? __fdiv_rn(1.0f, 1.0f + expf(-l)) : expf(fminf(l, 3.402823466e38f) - mx) * inv;
}

// The choice from 64-bit keys, in shared memory.  -> the id of choice `lane` (-1: none).
template <typename T>
__device__ __noinline__ int rt_choose64(const RouteParams& p, const T* row, double* key, double* gscore, int lane) {
    const double none = -INFINITY;
    double m = none;
    for (int e = lane; e < p.E; e += 32) m = fmax(m, (double)(rt_off(to_f32(row[e])) ? -INFINITY : fminf(to_f32(row[e]), 3.402823466e38f)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    double sum = 0;
    for (int e = lane; e < p.E; e += 32) {
        const float lf = to_f32(row[e]);
        const double l = fminf(lf, 3.402823466e38f);
        double k = none;
        if (!rt_off(lf)) {
            k = p.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m);
            sum += k;
        }
        key[e] = k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    for (int e = lane; e < p.E; e += 32) {
        double k = key[e];
        if (k != none) {
            if (!p.sigmoid) k /= sum;
            if (p.bias) k += (double)rt_bias(p, e);
        }
        key[e] = k;
    }
    __syncwarp();
    if (p.n_group > 1) {
        const int gs = p.E / p.n_group;
        double a = none, b = none;
        if (lane < p.n_group)
            for (int i = 0; i < gs; ++i) {
                const double k = key[lane * gs + i];
                if (k > a) { b = a; a = k; } else if (k > b) b = k;
            }
        const double g = a == none ? none : (p.top2 && b != none ? a + b : a);
        if (lane < p.n_group) gscore[lane] = g;
        __syncwarp();
        int before = 0;
        if (lane < p.n_group)
            for (int i = 0; i < p.n_group; ++i) before += gscore[i] > g || (gscore[i] == g && i < lane);
        if (lane < p.n_group && before >= p.topk_group)
            for (int i = 0; i < gs; ++i) key[lane * gs + i] = none;
        __syncwarp();
    }
    int mine = -1;
    for (int k = 0; k < p.top_k; ++k) {
        double best = none;
        int at = -1;
        for (int e = lane; e < p.E; e += 32)
            if (key[e] > best) { best = key[e]; at = e; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa >= 0 && (at < 0 || oa < at))) { best = ob; at = oa; }
        }
        if (at < 0) break;
        if (lane == k) mine = at;
        if (lane == (at & 31)) key[at] = none;
        __syncwarp();
    }
    return mine;
}

// One warp per token.
template <typename T, int PER>
__global__ void __launch_bounds__(RT_WARPS * 32) route_kernel(const RouteParams p) {
    extern __shared__ double rt_smem[];              // per warp: E 64-bit keys and the groups' scores
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * RT_WARPS + warp;
    if (t >= p.T) return;
    double* key64 = rt_smem + (long long)warp * (p.E + RT_MAX_GROUPS);
    float* skey = reinterpret_cast<float*>(key64);
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    float l[PER];
    rt_load<T, PER>(row, p.E, lane, p.vec, l);
    float mx = 0.0f, inv = 0.0f;
    if (!p.sigmoid) rt_softmax(l, &mx, &inv);
    uint32_t key[PER];
    const bool need_score = p.bias != nullptr || p.n_group > 1;
    bool close = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = lane * PER + j;
        float k = l[j];
        if (need_score && e < p.E) {
            k = rt_score(l[j], p.sigmoid, mx, inv);
            if (p.bias) k += rt_bias(p, e);
            if (l[j] == -INFINITY || !(k > -INFINITY)) k = -INFINITY;
            skey[e] = k;
        }
        key[j] = k == -INFINITY ? 0u : rt_order(p.bias ? k : l[j]);
    }
    if (p.n_group > 1) {
        __syncwarp();
        const int gs = p.E / p.n_group;
        float a = -INFINITY, b = -INFINITY;
        if (lane < p.n_group)
            for (int i = 0; i < gs; ++i) {
                const float k = skey[lane * gs + i];
                if (k > a) { b = a; a = k; } else if (k > b) b = k;
            }
        const float g = p.top2 && b > -INFINITY ? a + b : a;
        int before = 0;
        for (int i = 0; i < p.n_group; ++i) {
            const float o = __shfl_sync(0xffffffffu, g, i);
            before += o > g || (o == g && i < lane);
            // keys of two groups so close that their order needs 64 bits (both empty: the order does not matter)
            close |= lane < p.n_group && i != lane && o > -INFINITY && rt_close(o, g);
        }
        const unsigned keep = __ballot_sync(0xffffffffu, lane < p.n_group && before < p.topk_group);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = lane * PER + j;
            if (e < p.E && !((keep >> (e / gs)) & 1u)) key[j] = 0u;
        }
    }
    int mine = -1;
    float last = INFINITY;
    const int rounds = p.bias ? p.top_k + 1 : p.top_k;          // with a bias the best one left out is looked at too
    for (int k = 0; k < rounds; ++k) {
        uint32_t best = key[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < PER; ++j) if (key[j] > best) { best = key[j]; at = j; }
        const uint32_t m = __reduce_max_sync(0xffffffffu, best);
        if (m == 0u) break;
        const int winner = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
        const int e = __shfl_sync(0xffffffffu, lane * PER + at, winner);
        if (lane == k && k < p.top_k) mine = e;
        if (lane == winner) {
#pragma unroll
            for (int j = 0; j < PER; ++j) if (j == at) key[j] = 0u;
        }
        if (p.bias) {
            const float v = rt_unorder(m);
            close |= rt_close(v, last);
            last = v;
        }
    }
    if (need_score && __any_sync(0xffffffffu, close)) {
        __syncwarp();
        mine = rt_choose64<T>(p, row, key64, key64 + p.E, lane);
    }
    const float s = mine >= 0 ? rt_score(to_f32(row[mine]), p.sigmoid, mx, inv) : 0.0f;
    const float total = warp_sum(s) + 1e-20f;
    if (lane < p.top_k) {
        p.ids[(long long)t * p.top_k + lane] = mine;
        p.weights[(long long)t * p.top_k + lane] = (p.renorm ? __fdiv_rn(s, total) : s) * p.scale;
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

template <typename T, int PER>
__global__ void __launch_bounds__(RT_WARPS * 32) route_grad_kernel(const RouteGradParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * RT_WARPS + warp;
    if (t >= p.T) return;
    const T* row = static_cast<const T*>(p.logits) + t * p.stride;
    float l[PER];
    rt_load<T, PER>(row, p.E, lane, p.vec, l);
    float mx = 0.0f, inv = 0.0f;
    if (!p.sigmoid) rt_softmax(l, &mx, &inv);
    int id = -1;
    float g = 0.0f, s = 0.0f;
    if (lane < p.top_k) {
        id = __ldg(p.ids + (long long)t * p.top_k + lane);
        if (id >= p.E) id = -1;
        if (id >= 0) {
            float li = to_f32(row[id]);
            if (rt_off(li)) id = -1;
            else {
                s = rt_score(li, p.sigmoid, mx, inv);
                g = __ldg(p.grad + (long long)t * p.top_k + lane) * p.scale;
            }
        }
    }
    float dot = warp_sum(g * s);
    if (p.renorm) {
        const float total = warp_sum(s) + 1e-20f;
        g = id >= 0 ? __fdiv_rn(g - __fdiv_rn(dot, total), total) : 0.0f;
        dot = warp_sum(g * s);
    }
    float ds[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) ds[j] = 0.0f;
    for (int k = 0; k < p.top_k; ++k) {            // an expert that a token names twice gets both shares
        const int at = __shfl_sync(0xffffffffu, id, k) - lane * PER;
        const float v = __shfl_sync(0xffffffffu, g, k);
#pragma unroll
        for (int j = 0; j < PER; ++j) if (j == at) ds[j] += v;
    }
    T* out = static_cast<T*>(p.out) + (long long)t * p.E;
    constexpr int VL = PER < (int)(16 / sizeof(T)) ? PER : (int)(16 / sizeof(T));
#pragma unroll
    for (int j = 0; j < PER; j += VL) {
        struct alignas(sizeof(T) * VL) V { T v[VL]; } x;
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const float sc = rt_score(l[j + i], p.sigmoid, mx, inv);
            x.v[i] = from_f32<T>(p.sigmoid ? ds[j + i] * sc * (1.0f - sc) : sc * (ds[j + i] - dot));
        }
        if (p.vec) {
            if (lane * PER + j < p.E) *reinterpret_cast<V*>(out + lane * PER + j) = x;
        } else {
#pragma unroll
            for (int i = 0; i < VL; ++i) if (lane * PER + j + i < p.E) out[lane * PER + j + i] = x.v[i];
        }
    }
}

}  // namespace b200
