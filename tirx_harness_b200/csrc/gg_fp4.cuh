// m-grouped GEMM of 4-bit block-scaled operands: D_g = alpha_g * deq(A_g) * deq(B_g)^T.
//
// The block scales are applied inside the tensor core (tcgen05.mma kinds mxf4nvf4 and mxf4), which adds the exactly
// scaled products up in fp32; the factor alpha is applied to the sum.
//
// gg_fp4_pair_kernel: CTA pairs (cta_group::2), 256 x 256 tiles, 256 values of K per stage.  Per stage and CTA: 16 KB of A,
// 16 KB of B and 6 KB (nvfp4) or 3 KB (mxfp4) of scales -- those of its own 128 rows and of all 256 columns, which both
// CTAs' TMEM needs.  The scales come as the caller stores them, one contiguous piece per 128 rows and stage, and every
// stage has TMEM columns of its own for them, so that the barrier that hands the stage over also covers them.  One
// accumulator: two of 192 columns overlap the drain with the next tile's products but move 17 % more bytes per flop;
// 28672 x 4096 x 7168 in 32 groups took 524 us with them and 507 us with this, both before the row blocks were paired (see
// build_pair_list), under the power cap.  Two of 224 columns were not tried.
#pragma once

#include "fp4_ops.cuh"
#include "gg_fp8_mx.cuh"

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

// ------------------------------------------------------------------ PTX for 4-bit operands
// K = 64 values (32 bytes) per instruction.  NV: UE4M3 scales, four per row and instruction; MX: UE8M0, two.
template <bool NV>
__device__ __forceinline__ void umma_fp4_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t tmem_sfa,
                                              uint32_t tmem_sfb, uint32_t accumulate) {
    if (NV)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb) : "memory");
}
// instruction descriptor: e2m1 x e2m1, K-major operands, dense K = 64; sf_id: first of the scale bytes it uses (MX: 0 or 2)
template <bool NV>
__device__ __forceinline__ uint32_t make_idesc_fp4(int m, int n, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10)          // scale id of B; A, B format: e2m1
           | (static_cast<uint32_t>(n >> 3) << 17)        // N / 8
           | (NV ? 0u : 1u << 23)                         // scale format: UE4M3 / UE8M0
           | (static_cast<uint32_t>(m >> 7) << 27)        // M / 128
           | (sf_id << 29);                               // scale id of A
}

namespace f4 {
constexpr int BM = 128, BKB = 128;                        // rows per CTA; bytes of K per stage (256 values)
constexpr int THREADS = 384;
constexpr int TMEM_COLS = 512;
constexpr int TN = 256;                                   // columns of a tile
template <bool NV> struct Cfg {
    static constexpr int SF_CHUNK = NV ? 2048 : 1024;     // scales of 128 rows x 256 values
    static constexpr int A_BYTES = BM * BKB, B_BYTES = (TN / 2) * BKB;
    static constexpr int SF_BYTES = 3 * SF_CHUNK;         // this CTA's rows, the tile's columns (2 x 128)
    static constexpr int STAGES = NV ? 5 : 6;
    static constexpr int SFA_COLS = NV ? 16 : 8, SF_COLS = 3 * SFA_COLS;      // TMEM: the accumulator, then a stage's scales
    static_assert(TN + STAGES * SF_COLS <= TMEM_COLS);
    static constexpr int OFF_B = STAGES * A_BYTES;
    static constexpr int OFF_SF = OFF_B + STAGES * B_BYTES;
    static constexpr int OFF_BARS = OFF_SF + STAGES * SF_BYTES;
    static constexpr int OFF_PREFIX = OFF_BARS + 256;
    static constexpr int SMEM_BYTES = OFF_PREFIX + (gg::MAX_MASKED_GROUPS + 1) * 4 + 12 + 1024;
};
}  // namespace f4

// ---- schedule of the contiguous layout: which two 128-row blocks a pair multiplies at a time
// PairScheduler (pair_common.cuh) cuts the rows into fixed blocks of 256 and visits each once per group found in it, so that
// a group that begins in the middle of one costs a tile more.  Here the blocks of 128 rows are listed with the groups found in
// them, and neighbouring blocks of one group are paired from its first one on.  A last block without a partner leaves the
// second half of the tile empty: its rows are fetched from behind the matrix, which reads as zeros and moves no data.
// Up to 1024 (block, group) entries, built by every block for itself (M layout entries read once); larger ones and
// layouts with more groups per block take PairScheduler.
// 28672 rows in 32 ragged groups (4096 x 7168): 438 us with fixed blocks, 382 us paired.
constexpr int PAIR_LIST_CAP = 1024, PAIR_LIST_BLOCK_BITS = 11, PAIR_LIST_MAX_G = 1 << 20;

// list[i] = first block | group << 11 | (two blocks) << 31; returns the number of tiles, -1: too many.  Called by the whole
// block; `scratch`: 3 * 1024 ints.
__device__ __forceinline__ int build_pair_list(const GGFp4Params& p, int* list, int* scratch) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int rows_end = p.rows_used ? min(p.M, max(0, __ldg(p.rows_used))) : p.M;
    const int nb = (rows_end + 127) >> 7;
    if (nb > PAIR_LIST_CAP || p.G > PAIR_LIST_MAX_G) return -1;
    int* count = scratch;                            // groups in a block
    int* lowest = scratch + PAIR_LIST_CAP;           // the first of them, then where the block's entries begin
    int* entry = scratch + 2 * PAIR_LIST_CAP;        // block | group << 11
    auto load = [&](int b, int (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = b * 128 + j * 32 + lane;
            v[j] = r < rows_end ? __ldg(p.layout + r) : -1;
            if (v[j] < 0 || v[j] >= p.G) v[j] = INT_MAX;
        }
    };
    auto after = [&](const int (&v)[4], int g) {     // the lowest group above g, INT_MAX: none
        int m = INT_MAX;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (v[j] > g) m = min(m, v[j]);
        return __reduce_min_sync(0xffffffffu, m);
    };
    constexpr int AHEAD = 8;                         // blocks under way per warp
    for (int b0 = warp * AHEAD; b0 < nb; b0 += warps * AHEAD) {
        int v[AHEAD][4];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) load(b0 + k, v[k]);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (b0 + k >= nb) break;
            const int first = after(v[k], -1);
            int most = -1, n = first != INT_MAX;
#pragma unroll
            for (int j = 0; j < 4; ++j) if (v[k][j] != INT_MAX) most = max(most, v[k][j]);
            most = __reduce_max_sync(0xffffffffu, most);
            if (most != first)
                for (int g = first; g < most; ++n) g = after(v[k], g);
            if (lane == 0) { count[b0 + k] = n; lowest[b0 + k] = first; }
        }
    }
    __syncthreads();
    int total = 0;                                   // the same in every warp
    for (int base = 0; base < nb; base += 32) {
        const int b = base + lane, n = b < nb ? count[b] : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        const int at = total + incl - n;
        if ((base >> 5) % warps == warp) {
            if (n == 1 && at < PAIR_LIST_CAP) entry[at] = b | lowest[b] << PAIR_LIST_BLOCK_BITS;
            for (unsigned todo = __ballot_sync(0xffffffffu, n > 1 && at + n <= PAIR_LIST_CAP); todo; todo &= todo - 1) {
                const int i = __ffs(todo) - 1;
                int to = __shfl_sync(0xffffffffu, at, i), v[4];
                load(base + i, v);
                for (int g = after(v, -1); g != INT_MAX; g = after(v, g), ++to)
                    if (lane == 0) entry[to] = (base + i) | g << PAIR_LIST_BLOCK_BITS;
            }
        }
        total += __shfl_sync(0xffffffffu, incl, 31);
    }
    __syncthreads();
    if (total > PAIR_LIST_CAP) return -1;
    // pairs: an entry continues the one before if it is the next block of the same group; every second one of such a run begins a
    // tile.  Each warp works the whole list out, warp 0 writes it.
    int tiles = 0, run = 0;                          // run: where the run of the last entry so far begins
    for (int base = 0; base < total; base += 32) {
        const int i = base + lane;
        const bool in = i < total;
        const int e = in ? entry[i] : -1;
        const bool cont = in && i > 0 && entry[i - 1] + 1 == e;
        int start = in && !cont ? i : run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, start, o);
            if (lane >= o) start = max(start, u);
        }
        run = __shfl_sync(0xffffffffu, start, 31);
        const bool head = in && ((i - start) & 1) == 0;
        const unsigned heads = __ballot_sync(0xffffffffu, head);
        if (warp == 0 && head) {
            const bool two = i + 1 < total && e + 1 == entry[i + 1];
            list[tiles + __popc(heads & ((1u << lane) - 1u))] = (int)((uint32_t)e | (two ? 0x80000000u : 0u));
        }
        tiles += __popc(heads);
    }
    return tiles;
}

// Walks the list, columns fastest, like PairScheduler.
struct PairListScheduler {
    const GGFp4Params& p;
    const int* list;
    int t, total, n_blocks, stride, rank;
    __device__ __forceinline__ PairListScheduler(const GGFp4Params& p_, const int* list_, int tiles, int n_blocks_, int rank_)
        : p(p_), list(list_), t(blockIdx.x >> 1), total(tiles * n_blocks_), n_blocks(n_blocks_), stride(gridDim.x >> 1), rank(rank_) {}
    __device__ __forceinline__ bool next(Tile& tile) {
        if (t >= total) return false;
        const uint32_t e = (uint32_t)list[t / n_blocks];
        const int b = (int)(e & ((1u << PAIR_LIST_BLOCK_BITS) - 1u));
        tile.g = (int)((e & 0x7FFFFFFFu) >> PAIR_LIST_BLOCK_BITS);
        tile.n_blk = t % n_blocks;
        tile.m0 = (rank == 0 || (e & 0x80000000u) ? b + rank : p.a_tiles) * 128;
        tile.rows = 128;
        t += stride;
        return true;
    }
};

// One of the two schedules, decided per launch and block alike.
template <bool MASKED> struct Fp4Sched {
    bool listed;
    PairListScheduler l;
    PairScheduler<MASKED> s;
    __device__ __forceinline__ Fp4Sched(const GGFp4Params& p, const GGParams& sp, const int* table, int tiles, int lane, int rank)
        : listed(!MASKED && tiles >= 0), l(p, table, tiles, sp.num_n_blocks, rank), s(sp, table, lane, rank) {}
    __device__ __forceinline__ bool next(Tile& tile) {
        if (listed) return l.next(tile);
        if (!s.next(tile)) return false;
        if (MASKED && tile.rows == 0) tile.m0 = l.p.G * l.p.M;        // nothing in this half: read zeros from behind the matrix
        return true;
    }
};

template <bool NV, bool MASKED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(f4::THREADS, 1)
gg_fp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                   const __grid_constant__ CUtensorMap tmap_sfa, const __grid_constant__ CUtensorMap tmap_sfb,
                   const GGFp4Params p, const GGParams sp, int* status) {
    using namespace f4;
    using C = Cfg<NV>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    // [0,S) full (leader's used), [S,2S) empty, then tmem_full, tmem_empty (leader's used)
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
    int* prefix = reinterpret_cast<int*>(smem + C::OFF_PREFIX);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);       // a value the compiler knows to be warp-uniform
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t full_bar = smem_u32(bars), empty_bar = smem_u32(bars + STAGES);
    const uint32_t tfull_bar = smem_u32(bars + 2 * STAGES), tempty_bar = smem_u32(bars + 2 * STAGES + 1);
    const uint32_t leader_full_bar = map_to_cta(full_bar, 0), leader_tempty_bar = map_to_cta(tempty_bar, 0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        mbar_init(tfull_bar, 1);
        mbar_init(tempty_bar, 16);                    // the 16 epilogue warps of the pair
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
        tma_prefetch_desc(&tmap_sfa);
        tma_prefetch_desc(&tmap_sfb);
    }
    if (MASKED && warp == 3) {
        int running = 0;
        for (int base = 0; base < p.G; base += 32) {
            const int g = base + lane;
            int mm = g < p.G ? __ldg(p.layout + g) : 0;
            mm = mm < 0 ? 0 : (mm > p.M ? p.M : mm);
            const int blocks = (mm + 255) / 256;
            int incl = blocks;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (g < p.G) prefix[g] = running + incl - blocks;
            running += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) prefix[p.G] = running;
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_base_slot), TMEM_COLS);
        tmem_relinquish_pair();
    }
    int listed_tiles = -1;
    if (!MASKED) {
        listed_tiles = build_pair_list(p, prefix, reinterpret_cast<int*>(smem));
        fence_proxy_async_smem();                 // the ring's memory served as scratch; bulk copies write it from here on
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_base_slot;
    const int KB = (p.K + 255) / 256;
    // columns the pair multiplies for column tile n_blk: TN, or what is left of N rounded up to 16 (columns past N are
    // computed from whatever rows follow in B and never stored)
    auto tile_cols = [&](int n_blk) { const int left = (p.N - n_blk * TN + 15) & ~15; return left < TN ? left : TN; };

    if (warp < 4) {
        setmaxnreg_dec<72>();
        if (warp == 0) {
            // ------------------------------------------------ TMA producer (both CTAs)
            Fp4Sched<MASKED> sched(p, sp, prefix, listed_tiles, lane, rank);
            Tile tile;
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            while (ok && sched.next(tile)) {
                const int n0 = tile.n_blk * TN;
                const int b_row = tile.g * p.N + n0 + (int)rank * (tile_cols(tile.n_blk) >> 1);
                const int a_blk = !MASKED ? tile.m0 >> 7 : (tile.rows == 0 ? p.G * p.a_tiles : tile.g * p.a_tiles + ((tile.m0 - tile.g * p.M) >> 7));
                const int b_blk = tile.g * p.b_tiles + (n0 >> 7);
                for (int kb = 0; kb < KB; ++kb) {
                    ok = mbar_wait_warp(empty_bar + 8 * stage, phase ^ 1, abort_flag, status, STATUS_TIMEOUT_SMEM_EMPTY);
                    if (!ok) break;
                    if (elect_one_sync()) {
                        const uint32_t fb = leader_full_bar + 8 * stage;
                        constexpr int CW = C::SF_CHUNK / 8;              // 64-bit words of a chunk
                        if (rank == 0) mbar_arrive_expect_tx(full_bar + 8 * stage, 2 * (C::A_BYTES + C::B_BYTES + C::SF_BYTES));
                        tma_load_2d_pair(smem_u32(smem + stage * C::A_BYTES), &tmap_a, fb, kb * BKB, tile.m0);
                        tma_load_2d_pair(smem_u32(smem + C::OFF_B + stage * C::B_BYTES), &tmap_b, fb, kb * BKB, b_row);
                        const uint32_t sf = smem_u32(smem + C::OFF_SF + stage * C::SF_BYTES);
                        tma_load_1d_pair(sf, &tmap_sfa, fb, (a_blk * KB + kb) * CW);
                        tma_load_1d_pair(sf + C::SF_CHUNK, &tmap_sfb, fb, (b_blk * KB + kb) * CW);
                        tma_load_1d_pair(sf + 2 * C::SF_CHUNK, &tmap_sfb, fb, ((b_blk + 1) * KB + kb) * CW);
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                }
            }
            if (!ok) {                // unwinding: copies in flight get time to land before the CTA's memory goes
                const uint64_t t0 = globaltimer_ns();
                while (globaltimer_ns() - t0 < 1000000ull) {}
            }
        } else if (warp == 1 && rank == 0) {
            // ------------------------------------------------ MMA issuer (leader)
            Fp4Sched<MASKED> sched(p, sp, prefix, listed_tiles, lane, rank);
            Tile tile, next_tile;
            uint32_t stage = 0, phase = 0, acc_phase = 0;
            bool ok = true;
            const uint64_t adesc0 = make_smem_desc_sw128(smem_u32(smem));
            const uint64_t bdesc0 = make_smem_desc_sw128(smem_u32(smem + C::OFF_B));
            const uint64_t sdesc0 = make_sf_desc(smem_u32(smem + C::OFF_SF));
            bool have = sched.next(tile), have_next = false;
            while (ok && have) {
                ok = mbar_wait_warp(tempty_bar, acc_phase ^ 1, abort_flag, status, STATUS_TIMEOUT_TMEM_EMPTY);
                if (!ok) break;
                tc_fence_after();
                const uint32_t idesc = make_idesc_fp4<NV>(2 * BM, tile_cols(tile.n_blk), 0);
                for (int kb = 0; kb < KB; ++kb) {
                    ok = mbar_wait_warp(full_bar + 8 * stage, phase, abort_flag, status, STATUS_TIMEOUT_SMEM_FULL);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one_sync()) {
                        const uint32_t tsf = tmem_base + TN + stage * C::SF_COLS;
                        const uint64_t sd = sdesc0 + stage * (C::SF_BYTES >> 4);
                        constexpr int TILES = C::SFA_COLS / 4;
#pragma unroll
                        for (int j = 0; j < TILES; ++j) {
                            tmem_cp_sf_pair(tsf + 4 * j, sd + j * 32);
                            tmem_cp_sf_pair(tsf + C::SFA_COLS + 8 * j, sd + (C::SF_CHUNK >> 4) + j * 32);
                            tmem_cp_sf_pair(tsf + C::SFA_COLS + 8 * j + 4, sd + 2 * (C::SF_CHUNK >> 4) + j * 32);
                        }
                        const uint64_t adesc = adesc0 + stage * (C::A_BYTES >> 4), bdesc = bdesc0 + stage * (C::B_BYTES >> 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int w = NV ? j : j >> 1;
                            const uint32_t id = NV ? 0u : (uint32_t)(j & 1) * 2u;
                            umma_fp4_pair<NV>(tmem_base, adesc + 2 * j, bdesc + 2 * j, idesc | (id << 4) | (id << 29), tsf + 4 * w,
                                              tsf + C::SFA_COLS + 8 * w, kb > 0 || j > 0 ? 1u : 0u);
                        }
                        umma_commit_pair(empty_bar + 8 * stage, 3);
                        if (kb == KB - 1) umma_commit_pair(tfull_bar, 3);
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    if (kb == 0) have_next = sched.next(next_tile);
                }
                tile = next_tile;
                have = have_next;
                acc_phase ^= 1;
            }
        }
    } else {
        // ---------------------------------------------------- epilogue (both CTAs)
        setmaxnreg_inc<208>();
        constexpr int COLS = TN / 2, CHUNKS = COLS / 32;
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const int row_in_tile = quarter * 32 + lane;
        const int m_end = !MASKED && p.rows_used ? min(p.M, __ldg(p.rows_used)) : p.M;       // rows behind it are not written
        Fp4Sched<MASKED> sched(p, sp, prefix, listed_tiles, lane, rank);
        Tile tile;
        uint32_t acc_phase = 0;
        bool ok = true;
        while (ok && sched.next(tile)) {
            const int n0 = tile.n_blk * TN + half * COLS;
            const int row = tile.m0 + row_in_tile;
            const bool row_valid = MASKED ? row_in_tile < tile.rows : (row < m_end && __ldg(p.layout + row) == tile.g);
            const float alpha = p.alpha ? __ldg(p.alpha + tile.g * p.alpha_stride) : 1.0f;
            ok = mbar_wait_warp(tfull_bar, acc_phase, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL);
            if (!ok) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + half * COLS;
            uint32_t v[CHUNKS][32];
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) tmem_ld_32x32b_x32(taddr + c * 32, v[c]);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) tmem_ld_wait(v[c]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_tempty_bar);
            acc_phase ^= 1;
            if (!row_valid) continue;
            if (p.d_f32) {
                float* drow = static_cast<float*>(p.d) + (long long)row * p.ldd + n0;
#pragma unroll
                for (int j = 0; j < COLS; j += 4) {
                    if (n0 + j + 4 <= p.N)
                        *reinterpret_cast<float4*>(drow + j) =
                            make_float4(__uint_as_float(v[j / 32][j % 32]) * alpha, __uint_as_float(v[j / 32][j % 32 + 1]) * alpha,
                                        __uint_as_float(v[j / 32][j % 32 + 2]) * alpha, __uint_as_float(v[j / 32][j % 32 + 3]) * alpha);
                }
            } else {
                // one 32-byte sector per thread and store where the row is 32-byte aligned, else 16-byte stores
                __nv_bfloat16* drow = static_cast<__nv_bfloat16*>(p.d) + (long long)row * p.ldd + n0;
                const bool wide = (reinterpret_cast<uintptr_t>(drow) & 31u) == 0;
#pragma unroll
                for (int j = 0; j < COLS; j += 16) {
                    if (n0 + j < p.N) {
                        uint32_t o[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t* q = &v[(j + 2 * i) / 32][(j + 2 * i) % 32];
                            o[i] = cvt_bf16x2(pack_f32x2(__uint_as_float(q[0]) * alpha, __uint_as_float(q[1]) * alpha));
                        }
                        if (wide && n0 + j + 16 <= p.N) {
                            st_global_v8(drow + j, o);
                        } else {
                            if (n0 + j + 8 <= p.N) *reinterpret_cast<uint4*>(drow + j) = make_uint4(o[0], o[1], o[2], o[3]);
                            if (n0 + j + 16 <= p.N) *reinterpret_cast<uint4*>(drow + j + 8) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// ------------------------------------------------------------------ few rows per group
// gg_fp4_few_kernel: the weights' rows are the MMA's M (128 per tile), up to NT = 32 or 128 rows of a group its N, so a tile
// streams 128 rows of B over all of K and multiplies little in vain.  Bound by reading the weights from HBM: two blocks per
// SM (NT = 32) keep four 16 KB stages each under way (8 rows in 32 groups, 4096 x 7168: 82 us, 6.4 TB/s; one row in 8 groups:
// 23 us).  Two accumulators: a tile is stored while the next one is multiplied.  Blocks come in clusters of CLUSTER.  Where
// there are more tiles than clusters, or K is short, every block takes tiles of its own; else the blocks of a cluster take
// a part of K each and add their sums up, always in the same order, through each other's shared memory (one row, 4096 x
// 7168: 7.6 us instead of 11.2).  Clusters of two, of which 74 fit; clusters of four fit on 132 of the 148 SMs only, which
// costs 32 groups of 8 rows 104 us instead of 82, and serve calls that cannot have more than 32 tiles.
namespace ff {
constexpr int BKB = 128, THREADS = 256, ACCS = 2;
constexpr int FOUR_MAX_TILES = 32;
constexpr int LIST_CAP = 1024;               // (group, chunk of rows) entries: the host sees to it that there are no more,
constexpr int MAX_ROWS = 1024;               // nor more rows in the contiguous layout
template <bool NV, int NT> struct Cfg {
    static constexpr int SF_CHUNK = NV ? 2048 : 1024;
    static constexpr int W_BYTES = 128 * BKB, X_BYTES = NT * BKB;
    static constexpr int STAGE = W_BYTES + X_BYTES + 2 * SF_CHUNK;
    static constexpr int STAGES = NT == 32 ? 4 : 5;
    static constexpr int BLOCKS_PER_SM = NT == 32 ? 2 : 1;
    // a stage of K takes 0.25 us, adding the blocks' sums up 1.7 us (NT = 32) or 2.5 us: where K is shorter it is not shared
    static constexpr int SPLIT_MIN_KB = NT == 32 ? 16 : 24;
    static constexpr int SF_COLS = NV ? 16 : 8;                  // scale columns of one operand and stage
    static constexpr int COLS = ACCS * NT + STAGES * 2 * SF_COLS, TMEM_COLS = COLS > 256 ? 512 : (COLS > 128 ? 256 : 128);
    static constexpr int OFF_X = STAGES * W_BYTES;
    static constexpr int OFF_SF = OFF_X + STAGES * X_BYTES;
    static constexpr int OFF_BARS = OFF_SF + STAGES * 2 * SF_CHUNK;
    static constexpr int OFF_LIST = OFF_BARS + 256;
    static constexpr int SMEM_BYTES = OFF_LIST + LIST_CAP * 4 + 1024;
    static_assert(COLS <= 512 && BLOCKS_PER_SM * TMEM_COLS <= 512, "accumulators and scales must fit TMEM");
    static_assert(STAGES * STAGE >= NT / 8 * 128 * 12 * 4, "the ring's memory holds the sums of a cluster's blocks for one block's rows");
};
}  // namespace ff

template <bool NV>
__device__ __forceinline__ void umma_fp4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t tmem_sfa, uint32_t tmem_sfb,
                                         uint32_t accumulate) {
    if (NV)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb) : "memory");
}

// S accumulator columns (8 or 16), i.e. rows of d, of this warp's 32 lanes, i.e. columns of d
template <int S> __device__ __forceinline__ void few_load(uint32_t taddr, uint32_t (&v)[S]) {
    static_assert(S == 8 || S == 16, "");
    if constexpr (S == 8) {
        tmem_ld_32x32b_x8(taddr, v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])::"memory");
    } else {
        tmem_ld_32x32b_x16(taddr, v);
        tmem_ld_wait(v);
    }
}
// S rows of one column of d: row j, where bit j of `rows` is set, at d + j * ldd
template <typename T, int S>
__device__ __forceinline__ void few_store(T* d, long long ldd, unsigned rows, const uint32_t (&v)[S], float alpha) {
#pragma unroll
    for (int j = 0; j < S; ++j, d += ldd)
        if ((rows >> j) & 1u) *d = from_f32<T>(__uint_as_float(v[j]) * alpha);
}

template <bool NV, int NT, int CLUSTER>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(ff::THREADS, 2)
gg_fp4_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const GGFp4Params p, int x_box_rows,
                  int* status) {
    using namespace ff;
    using C = Cfg<NV, NT>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);          // full[S], empty[S], tmem_full[2], tmem_empty[2]
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
    int* list = reinterpret_cast<int*>(smem + C::OFF_LIST);                    // group | chunk of NT rows << 20, where it has rows
    volatile int* list_len = reinterpret_cast<volatile int*>(tmem_base_slot + 2);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t full_bar = smem_u32(bars), empty_bar = smem_u32(bars + STAGES);
    const uint32_t tfull_bar = smem_u32(bars + 2 * STAGES), tempty_bar = smem_u32(bars + 2 * STAGES + 2);
    const int rows_end = !p.masked && p.rows_used ? min(p.M, __ldg(p.rows_used)) : p.M;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        for (int a = 0; a < ACCS; ++a) {
            mbar_init(tfull_bar + 8 * a, 1);
            mbar_init(tempty_bar + 8 * a, 4);
        }
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmap_w);
        tma_prefetch_desc(&tmap_x);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_base_slot), C::TMEM_COLS);
        tmem_relinquish();
    }
    int* groups = reinterpret_cast<int*>(smem);            // contiguous layout: the rows' groups, in the ring's memory for now
    if (!p.masked) {
        for (int r = threadIdx.x; r < p.M; r += THREADS) groups[r] = r < rows_end ? __ldg(p.layout + r) : -1;
        __syncthreads();
    }
    if (warp == 2) {
        int n = 0;
        if (p.masked) {
            for (int base = 0; base < p.G; base += 32) {
                const int g = base + lane, rows = g < p.G ? min(p.M, max(0, __ldg(p.layout + g))) : 0, chunks = (rows + NT - 1) / NT;
                int incl = chunks;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                for (int c = 0; c < chunks; ++c) list[n + incl - chunks + c] = g | c << 20;
                n += __shfl_sync(0xffffffffu, incl, 31);
            }
        } else {
            for (int row0 = 0; row0 < p.M; row0 += NT) {
                // the distinct groups of the chunk's rows, ascending
                int vals[NT / 32];
#pragma unroll
                for (int j = 0; j < NT / 32; ++j) {
                    const int r = row0 + lane + 32 * j;
                    vals[j] = r < p.M ? groups[r] : -1;
                }
                for (int after = -1;; ++n) {
                    int best = INT_MAX;
#pragma unroll
                    for (int j = 0; j < NT / 32; ++j)
                        if (vals[j] > after && vals[j] < p.G && vals[j] < best) best = vals[j];
                    best = __reduce_min_sync(0xffffffffu, best);
                    if (best == INT_MAX) break;
                    if (lane == 0) list[n] = best | (row0 / NT) << 20;
                    after = best;
                }
            }
        }
        if (lane == 0) *list_len = n;
    }
    fence_proxy_async_smem();                     // bulk copies write the ring from here on
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_base_slot;
    const int KB = (p.K + 255) / 256, n_tiles = (p.N + 127) / 128;
    const int tiles = *list_len * n_tiles, clusters = gridDim.x / CLUSTER;
    const int rank = (int)cluster_ctarank(), cluster = blockIdx.x / CLUSTER;
    // few tiles: one per cluster, a part of K per block; else one after the other per block, spread over the clusters first
    const bool split = tiles <= clusters && KB >= C::SPLIT_MIN_KB;
    const int first = split ? cluster : rank * clusters + cluster, step = gridDim.x;
    const int kb0 = split ? KB * rank / CLUSTER : 0, kb1 = split ? KB * (rank + 1) / CLUSTER : KB;

    if (warp == 0) {
        // ------------------------------------------------ producer
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (int t = first; ok && t < tiles; t += step) {
            const int e = list[t / n_tiles], g = e & 0xFFFFF, chunk = e >> 20, nt = t % n_tiles;
            const int w_row = g * p.N + nt * 128, x_row = (p.masked ? g * p.M : 0) + chunk * NT;
            const uint8_t* sfw = p.sfb + ((long long)g * p.b_tiles + nt) * KB * C::SF_CHUNK;
            // (NT = 32 has one chunk)
            const uint8_t* sfx = p.sfa + ((p.masked ? (long long)g * p.a_tiles : 0) + chunk) * KB * C::SF_CHUNK;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait_warp(empty_bar + 8 * stage, phase ^ 1, abort_flag, status, STATUS_TIMEOUT_SMEM_EMPTY);
                if (!ok) break;
                if (elect_one_sync()) {
                    const uint32_t fb = full_bar + 8 * stage, sf = smem_u32(smem + C::OFF_SF + stage * 2 * C::SF_CHUNK);
                    mbar_arrive_expect_tx(fb, C::W_BYTES + x_box_rows * BKB + 2 * C::SF_CHUNK);
                    tma_load_2d(smem_u32(smem + stage * C::W_BYTES), &tmap_w, fb, kb * BKB, w_row);
                    tma_load_2d(smem_u32(smem + C::OFF_X + stage * C::X_BYTES), &tmap_x, fb, kb * BKB, x_row);
                    bulk_load(sf, sfw + (long long)kb * C::SF_CHUNK, C::SF_CHUNK, fb);
                    bulk_load(sf + C::SF_CHUNK, sfx + (long long)kb * C::SF_CHUNK, C::SF_CHUNK, fb);
                }
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
        }
        if (!ok) {                // unwinding: copies in flight get time to land before the block's memory goes
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 1000000ull) {}
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
        bool ok = true;
        const uint64_t wdesc0 = make_smem_desc_sw128(smem_u32(smem)), xdesc0 = make_smem_desc_sw128(smem_u32(smem + C::OFF_X));
        const uint64_t sdesc0 = make_sf_desc(smem_u32(smem + C::OFF_SF));
        const uint32_t idesc = make_idesc_fp4<NV>(128, NT, 0);
        for (int t = first; ok && t < tiles; t += step) {
            ok = mbar_wait_warp(tempty_bar + 8 * acc, acc_phase ^ 1, abort_flag, status, STATUS_TIMEOUT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait_warp(full_bar + 8 * stage, phase, abort_flag, status, STATUS_TIMEOUT_SMEM_FULL);
                if (!ok) break;
                tc_fence_after();
                if (elect_one_sync()) {
                    const uint32_t sfw = tmem_base + ACCS * NT + stage * 2 * C::SF_COLS, sfx = sfw + C::SF_COLS;
                    const uint64_t sd = sdesc0 + stage * (2 * C::SF_CHUNK >> 4);
#pragma unroll
                    for (int j = 0; j < C::SF_COLS / 4; ++j) {
                        tmem_cp_sf(sfw + 4 * j, sd + j * 32);
                        tmem_cp_sf(sfx + 4 * j, sd + (C::SF_CHUNK >> 4) + j * 32);
                    }
                    const uint64_t wd = wdesc0 + stage * (C::W_BYTES >> 4), xd = xdesc0 + stage * (C::X_BYTES >> 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int w = NV ? j : j >> 1;
                        const uint32_t id = NV ? 0u : (uint32_t)(j & 1) * 2u;
                        umma_fp4<NV>(tmem_base + acc * NT, wd + 2 * j, xd + 2 * j, idesc | (id << 4) | (id << 29), sfw + 4 * w, sfx + 4 * w,
                                     kb > kb0 || j > 0 ? 1u : 0u);
                    }
                    umma_commit(empty_bar + 8 * stage);
                    if (kb == kb1 - 1) umma_commit(tfull_bar + 8 * acc);
                }
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
            if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
        }
    }
    // ---------------------------------------------------- epilogue: thread = column of d, register = row
    const int ew = warp - 4;                       // TMEM lane quarter (warp % 4)
    // Rows are taken S at a time: the code is short, which is what a call of one tile waits for (unrolled over 32 rows, the
    // instruction fetches alone took 2 us), and a call with few rows runs through it once.
    constexpr int S = NT == 32 ? 8 : 16;
    // which of the S rows from row0 on belong to group g
    auto rows_of = [&](int g, int row0) -> unsigned {
        if (p.masked) {
            const int left = min(p.M, __ldg(p.layout + g)) - row0;
            return left >= S ? (1u << S) - 1u : (left > 0 ? (1u << left) - 1u : 0u);
        }
        return __ballot_sync(0xffffffffu, lane < S && row0 + lane < rows_end && __ldg(p.layout + row0 + lane) == g);
    };
    auto alpha_of = [&](int g) { return p.alpha ? __ldg(p.alpha + g * p.alpha_stride) : 1.0f; };
    auto put = [&](int g, int row0, int n, unsigned rows, const uint32_t (&v)[S], float alpha) {
        const long long o = ((p.masked ? (long long)g * p.M : 0) + row0) * p.ldd + n;
        if (n >= p.N) rows = 0u;
        if (p.d_f32) few_store(static_cast<float*>(p.d) + o, p.ldd, rows, v, alpha);
        else few_store(static_cast<__nv_bfloat16*>(p.d) + o, p.ldd, rows, v, alpha);
    };
    if (warp >= 4 && !split) {
        uint32_t acc = 0, acc_phase = 0;
        for (int t = first; t < tiles; t += step) {
            const int e = list[t / n_tiles], g = e & 0xFFFFF, row0 = (e >> 20) * NT, n = (t % n_tiles) * 128 + ew * 32 + lane;
            const float alpha = alpha_of(g);
            if (!mbar_wait_warp(tfull_bar + 8 * acc, acc_phase, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL)) break;
            tc_fence_after();
#pragma unroll 1
            for (int w = 0; w < NT; w += S) {
                const unsigned rows = rows_of(g, row0 + w);
                if (rows == 0u) continue;
                uint32_t v[S];
                few_load(tmem_base + (uint32_t(ew * 32) << 16) + acc * NT + w, v);
                put(g, row0 + w, n, rows, v, alpha);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar + 8 * acc);
            if (++acc == ACCS) { acc = 0; acc_phase ^= 1; }
        }
    }
    if (split) {
        // S rows at a time belong to the blocks of the cluster in turn, which finish them
        const bool work = first < tiles;
        const int e = work ? list[first / n_tiles] : 0, g = e & 0xFFFFF, row0 = (e >> 20) * NT;
        const int c = ew * 32 + lane, n = (work ? (first % n_tiles) * 128 : 0) + c;
        const uint32_t acc = tmem_base + (uint32_t(ew * 32) << 16);
        if (warp >= 4 && work) mbar_wait_warp(tfull_bar, 0, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL);
        __syncwarp();
        // every block of the cluster has read all of its stages: their memory takes the other blocks' sums of the rows that a
        // block is to finish, [rank][S rows][column][row] (a thread sends its rows 16 bytes at a time; the distance between
        // columns keeps the banks apart)
        constexpr int PITCH = S + 4;
        auto slot = [&](int from, int w) { return ((from * (NT / CLUSTER / S) + w / S / CLUSTER) * 128 + c) * PITCH; };
        cluster_sync_all();
        if (warp >= 4 && work) {
            tc_fence_after();
#pragma unroll 1
            for (int w = 0; w < NT; w += S) {
                const unsigned rows = rows_of(g, row0 + w);
                const int owner = w / S % CLUSTER;
                if (rows == 0u || owner == rank) continue;
                uint32_t v[S];
                few_load(acc + w, v);
                const uint32_t dst = map_to_cta(smem_u32(smem), owner) + slot(rank, w) * 4;
#pragma unroll
                for (int j = 0; j < S; j += 4)
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};"
                                 ::"r"(dst + j * 4), "r"(v[j]), "r"(v[j + 1]), "r"(v[j + 2]), "r"(v[j + 3]) : "memory");
            }
        }
        __syncwarp();
        cluster_sync_all();
        if (warp >= 4 && work) {
            const float alpha = alpha_of(g);
#pragma unroll 1
            for (int w = rank * S; w < NT; w += CLUSTER * S) {
                const unsigned rows = rows_of(g, row0 + w);
                if (rows == 0u) continue;
                uint32_t v[S];
                few_load(acc + w, v);
                float sum[S];
#pragma unroll
                for (int j = 0; j < S; ++j) sum[j] = 0.0f;
#pragma unroll 1
                for (int r = 0; r < CLUSTER; ++r) {        // in the order of the ranks
                    const float4* part = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + slot(r, w));
#pragma unroll
                    for (int j = 0; j < S; j += 4) {
                        float4 x = make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
                        if (r != rank) x = part[j / 4];
                        sum[j] += x.x; sum[j + 1] += x.y; sum[j + 2] += x.z; sum[j + 3] += x.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < S; ++j) v[j] = __float_as_uint(sum[j]);
                put(g, row0 + w, n, rows, v, alpha);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

}  // namespace b200
