// Host side of the norm, routing and 4-bit entry points: validation and launches.  Included by b200moe.cu, whose error
// reporting and device table it uses.
#pragma once

namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool float_dtype(int d) { return d == MOE_DTYPE_BF16 || d == MOE_DTYPE_F32 || d == MOE_DTYPE_F16; }
// Most rows of a call whose kernels count rows and blocks of up to 128 of them in 32 bits.
constexpr int32_t MAX_ROWS_32 = 0x7FFFFFFF - 127;
inline int dtype_bytes(int d) { return d == MOE_DTYPE_F32 ? 4 : 2; }

// f(a value of the element type)
template <typename F>
void with_dtype(int dtype, F f) {
    if (dtype == MOE_DTYPE_BF16) f(__nv_bfloat16{});
    else if (dtype == MOE_DTYPE_F16) f(__half{});
    else f(float{});
}

// Raises a kernel's dynamic shared memory limit, once per device; `done` belongs to the kernel.
template <typename K>
int raise_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));              // below 64: device_info has been called
    const uint64_t bit = 1ull << dev;
    if (done.load(std::memory_order_acquire) & bit) return MOE_OK;
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
    return MOE_OK;
}

int check_norm(int32_t T, int32_t H, int32_t dtype, int32_t w_dtype) {
    if (T < 0 || H <= 0 || H % 8 || H > NORM_MAX_H)
        return fail(MOE_ERR_INVALID, "T=%d must be non-negative and H=%d a multiple of 8 in [8, %d]", T, H, NORM_MAX_H);
    if (!float_dtype(dtype) || (w_dtype != dtype && w_dtype != MOE_DTYPE_F32))
        return fail(MOE_ERR_INVALID, "dtype must be bf16, f16 or f32, and w_dtype the same or f32");
    return MOE_OK;
}
int check_rows(const char* name, const void* p, int64_t stride, int32_t H) {
    if (!p) return fail(MOE_ERR_INVALID, "%s must be non-NULL", name);
    if (!aligned16(p) || stride < H || stride % 8)
        return fail(MOE_ERR_INVALID, "%s must be 16-byte aligned with a row stride >= H that is a multiple of 8", name);
    return MOE_OK;
}

// Threads and 8-column pieces per thread.  Two pieces: what a row costs every warp (the sum over the block, the wait, its
// scalars) is shared by more columns than with one -- 16384 x 2048 bf16 forward 44 us against 50, backward 47 against 56 --
// and four need too many registers (46 and 51 us); they serve rows that 512 threads cannot hold otherwise.
struct NormShape { int threads, pieces; };
NormShape norm_shape(int H) {
    const int n8 = H / 8;
    NormShape s;
    s.pieces = n8 <= 2 * NORM_MAX_THREADS ? 2 : 4;
    s.threads = ((n8 + s.pieces - 1) / s.pieces + 31) / 32 * 32;
    return s;
}

// Blocks per SM and rows of the ring: as many threads as the registers allow (two blocks of 448 threads forward, one
// backward), and up to four rows each, which is several times the 45 KB per SM that cover memory's latency.
struct NormPlan { int per_sm, stages; size_t smem; };
NormPlan norm_plan(NormShape s, size_t stage_bytes, int threads_per_sm, int most_per_sm) {
    constexpr size_t room = 200 * 1024;
    NormPlan n;
    n.per_sm = threads_per_sm / s.threads;
    if (n.per_sm > most_per_sm) n.per_sm = most_per_sm;
    while (n.per_sm > 1 && (size_t)n.per_sm * (2 * stage_bytes + NORM_HEAD_BYTES) > room) --n.per_sm;
    if (n.per_sm < 1) n.per_sm = 1;
    n.stages = NORM_MAX_STAGES;
    while (n.stages > 1 && (size_t)n.per_sm * (n.stages * stage_bytes + NORM_HEAD_BYTES) > room) --n.stages;
    n.smem = NORM_HEAD_BYTES + n.stages * stage_bytes;
    return n;
}

constexpr int NORM_GRAD_THREADS = 768, NORM_GRAD_PER_SM = 12;         // per SM: threads, and blocks at most
// rows of fp32 that the blocks' shares of dw may take
int norm_grad_parts(int H) {
    const int per_sm = NORM_GRAD_THREADS / norm_shape(H).threads;
    return 160 * (per_sm < 1 ? 1 : (per_sm > NORM_GRAD_PER_SM ? NORM_GRAD_PER_SM : per_sm));
}

template <typename T, typename W, int CH>
int launch_norm_ch(NormParams p, NormShape s, DeviceInfo* di, cudaStream_t st) {
    const NormPlan n = norm_plan(s, (size_t)p.H * sizeof(T) * (p.residual ? 2 : 1), 1024, 24);
    p.stages = n.stages; p.status = di->status;
    const int grid = p.T < n.per_sm * di->num_sms ? p.T : n.per_sm * di->num_sms;
    static std::atomic<uint64_t> done{0};
    if (int rc = raise_smem(rms_norm_quant_kernel<T, W, CH>, 227 * 1024, done)) return rc;
    rms_norm_quant_kernel<T, W, CH><<<grid, s.threads, n.smem, st>>>(p);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}
template <typename T, typename W>
int launch_norm(const NormParams& p, NormShape s, DeviceInfo* di, cudaStream_t st) {
    if (s.pieces == 2) return launch_norm_ch<T, W, 2>(p, s, di, st);
    return launch_norm_ch<T, W, 4>(p, s, di, st);
}
template <typename T, typename W, int CH>
int launch_norm_grad_ch(NormGradParams p, float* dw, NormShape s, DeviceInfo* di, cudaStream_t st) {
    const NormPlan n = norm_plan(s, (size_t)p.H * sizeof(T) * (p.dh ? 3 : 2), NORM_GRAD_THREADS, NORM_GRAD_PER_SM);
    p.stages = n.stages; p.status = di->status;
    int grid = n.per_sm * di->num_sms;
    if (grid > norm_grad_parts(p.H)) grid = norm_grad_parts(p.H);
    if (grid > p.T) grid = p.T;
    static std::atomic<uint64_t> done{0};
    if (int rc = raise_smem(rms_norm_grad_kernel<T, W, CH>, 227 * 1024, done)) return rc;
    rms_norm_grad_kernel<T, W, CH><<<grid, s.threads, n.smem, st>>>(p);
    CUDA_TRY(cudaGetLastError());
    CUDA_TRY(launch_pdl(rms_norm_dw_kernel, dim3((p.H + 31) / 32), dim3(1024), 0, st, (const float*)p.partial, dw, grid, p.H));
    return MOE_OK;
}
template <typename T, typename W>
int launch_norm_grad(const NormGradParams& p, float* dw, NormShape s, DeviceInfo* di, cudaStream_t st) {
    if (s.pieces == 2) return launch_norm_grad_ch<T, W, 2>(p, dw, s, di, st);
    return launch_norm_grad_ch<T, W, 4>(p, dw, s, di, st);
}

int check_route(int32_t T, int32_t E, int32_t top_k, int32_t dtype, int32_t score, int64_t stride) {
    if (T < 0 || T > MAX_ROWS_32 || E <= 0 || E > RT_MAX_E)
        return fail(MOE_ERR_INVALID, "T=%d must be in [0, %d] and E=%d in [1, %d]", T, MAX_ROWS_32, E, RT_MAX_E);
    if (top_k <= 0 || top_k > 32 || top_k > E) return fail(MOE_ERR_INVALID, "top_k=%d must be in [1, min(32, E)]", top_k);
    if (!float_dtype(dtype)) return fail(MOE_ERR_INVALID, "dtype must be bf16, f16 or f32");
    if (score != MOE_SCORE_SOFTMAX && score != MOE_SCORE_SIGMOID) return fail(MOE_ERR_INVALID, "score must be MOE_SCORE_SOFTMAX or MOE_SCORE_SIGMOID");
    if (stride < E) return fail(MOE_ERR_INVALID, "stride=%lld must be >= E", (long long)stride);
    return MOE_OK;
}
// whole 16-byte pieces of a row can be read (and written, in a dense output) wherever a lane's experts begin
bool route_vec(const void* p, int64_t stride, int32_t E, int32_t dtype) {
    const int n = 16 / dtype_bytes(dtype);
    return aligned16(p) && stride % n == 0 && E % n == 0;
}

// consecutive experts that a lane holds
int route_per_lane(int E) { return E <= 128 ? 4 : (E <= 256 ? 8 : (E <= 512 ? 16 : 32)); }

template <typename T>
void launch_route(const RouteParams& p, size_t smem, cudaStream_t st) {
    const int grid = (p.T + RT_WARPS - 1) / RT_WARPS, block = RT_WARPS * 32;
    if (p.E <= 128) route_kernel<T, 4><<<grid, block, smem, st>>>(p);
    else if (p.E <= 256) route_kernel<T, 8><<<grid, block, smem, st>>>(p);
    else if (p.E <= 512) route_kernel<T, 16><<<grid, block, smem, st>>>(p);
    else route_kernel<T, 32><<<grid, block, smem, st>>>(p);
}
template <typename T>
void launch_route_grad(const RouteGradParams& p, cudaStream_t st) {
    const int grid = (p.T + RT_WARPS - 1) / RT_WARPS, block = RT_WARPS * 32;
    if (p.E <= 128) route_grad_kernel<T, 4><<<grid, block, 0, st>>>(p);
    else if (p.E <= 256) route_grad_kernel<T, 8><<<grid, block, 0, st>>>(p);
    else if (p.E <= 512) route_grad_kernel<T, 16><<<grid, block, 0, st>>>(p);
    else route_grad_kernel<T, 32><<<grid, block, 0, st>>>(p);
}

template <typename T>
void launch_quant_fp4(const Fp4QuantParams& p, bool nv, bool silu, bool by_row, dim3 grid, cudaStream_t st) {
    if (by_row && nv) quant_fp4_kernel<T, true, false, true><<<grid, FP4_QUANT_THREADS, 0, st>>>(p);
    else if (by_row) quant_fp4_kernel<T, false, false, true><<<grid, FP4_QUANT_THREADS, 0, st>>>(p);
    else if (nv && silu) quant_fp4_kernel<T, true, true, false><<<grid, FP4_QUANT_THREADS, 0, st>>>(p);
    else if (nv) quant_fp4_kernel<T, true, false, false><<<grid, FP4_QUANT_THREADS, 0, st>>>(p);
    else if (silu) quant_fp4_kernel<T, false, true, false><<<grid, FP4_QUANT_THREADS, 0, st>>>(p);
    else quant_fp4_kernel<T, false, false, false><<<grid, FP4_QUANT_THREADS, 0, st>>>(p);
}

// 1-D array of scale tiles as 64-bit words, box = one chunk (the scales of 128 rows x 256 values)
int encode_scale_chunks(CUtensorMap* map, const void* base, uint64_t bytes, uint32_t chunk) {
    auto fn = get_encode_fn();
    if (!fn) return fail(MOE_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[1] = {bytes / 8};
    cuuint64_t strides[1] = {0};
    cuuint32_t box[1] = {chunk / 8};
    cuuint32_t estr[1] = {1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 1, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MOE_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed with CUresult %d", (int)r);
    return MOE_OK;
}

template <bool NV, bool MASKED>
int launch_fp4_pair(const GGFp4Params& p, long long rows_total, DeviceInfo* di, cudaStream_t st) {
    using C = f4::Cfg<NV>;
    CUtensorMap ta, tb, tsa, tsb;
    int rc;
    const uint64_t kt = (uint64_t)p.kt * 512;
    if ((rc = encode_fp8_kmajor(&ta, p.a, (uint64_t)rows_total, (uint64_t)p.K / 2, f4::BM)) != MOE_OK) return rc;
    if ((rc = encode_fp8_kmajor(&tb, p.b, (uint64_t)p.G * p.N, (uint64_t)p.K / 2, f4::TN / 2)) != MOE_OK) return rc;
    if ((rc = encode_scale_chunks(&tsa, p.sfa, (uint64_t)(MASKED ? p.G : 1) * p.a_tiles * kt, C::SF_CHUNK)) != MOE_OK) return rc;
    if ((rc = encode_scale_chunks(&tsb, p.sfb, (uint64_t)p.G * p.b_tiles * kt, C::SF_CHUNK)) != MOE_OK) return rc;
    GGParams sp = {};
    sp.layout = p.layout; sp.rows_used = p.rows_used; sp.G = p.G; sp.M = p.M; sp.N = p.N;
    sp.num_n_blocks = (p.N + f4::TN - 1) / f4::TN;
    // row blocks that sorted rows can fill (more tiles than this only make the pairs take more than one each)
    const long long blocks = MASKED ? (long long)p.G * ((p.M + 255) / 256) : (p.M + 255) / 256 + (p.G < p.M ? p.G : p.M) - 1;
    const long long tiles = blocks * sp.num_n_blocks;
    const int pairs = (int)(tiles < di->max_pairs ? tiles : di->max_pairs);
    static std::atomic<uint64_t> done{0};
    if ((rc = raise_smem(gg_fp4_pair_kernel<NV, MASKED>, C::SMEM_BYTES, done)) != MOE_OK) return rc;
    gg_fp4_pair_kernel<NV, MASKED><<<2 * pairs, f4::THREADS, C::SMEM_BYTES, st>>>(ta, tb, tsa, tsb, p, sp, di->status);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}
template <bool NV>
int launch_fp4_pair_layout(const GGFp4Params& p, long long rows_total, DeviceInfo* di, cudaStream_t st) {
    return p.masked ? launch_fp4_pair<NV, true>(p, rows_total, di, st) : launch_fp4_pair<NV, false>(p, rows_total, di, st);
}

// the most (group, chunk of NT rows) that can have rows
long long fp4_few_entries(const GGFp4Params& p, int NT) {
    const long long chunks = (p.M + NT - 1) / NT;
    if (p.masked) return p.G * chunks;
    // a chunk has at most NT groups; sorted rows change groups G - 1 times at most, but they need not be sorted
    return chunks * (p.G < NT ? p.G : NT) < p.M ? chunks * (p.G < NT ? p.G : NT) : p.M;
}

template <bool NV, int NT, int CLUSTER>
int launch_fp4_few_clusters(const GGFp4Params& p, long long rows_total, long long tiles, DeviceInfo* di, cudaStream_t st) {
    using C = ff::Cfg<NV, NT>;
    CUtensorMap tw, tx;
    int rc;
    // no more rows than there are: the others of the stage keep whatever it held, and their products are not stored
    const int box = NT > 32 ? NT : (p.M <= 8 ? 8 : (p.M <= 16 ? 16 : 32));
    if ((rc = encode_fp8_kmajor(&tw, p.b, (uint64_t)p.G * p.N, (uint64_t)p.K / 2, 128)) != MOE_OK) return rc;
    if ((rc = encode_fp8_kmajor(&tx, p.a, (uint64_t)rows_total, (uint64_t)p.K / 2, box)) != MOE_OK) return rc;
    static std::atomic<uint64_t> done{0};
    if ((rc = raise_smem(gg_fp4_few_kernel<NV, NT, CLUSTER>, C::SMEM_BYTES, done)) != MOE_OK) return rc;
    const long long fit = (long long)C::BLOCKS_PER_SM * di->num_sms / CLUSTER;
    const int clusters = (int)(tiles < fit ? tiles : fit);
    gg_fp4_few_kernel<NV, NT, CLUSTER><<<clusters * CLUSTER, ff::THREADS, C::SMEM_BYTES, st>>>(tw, tx, p, box, di->status);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}
template <bool NV, int NT>
int launch_fp4_few(const GGFp4Params& p, long long rows_total, DeviceInfo* di, cudaStream_t st) {
    // the most tiles that can come: the groups with rows are known on the device only
    const long long tiles = fp4_few_entries(p, NT) * ((p.N + 127) / 128);
    return tiles <= ff::FOUR_MAX_TILES ? launch_fp4_few_clusters<NV, NT, 4>(p, rows_total, tiles, di, st)
                                       : launch_fp4_few_clusters<NV, NT, 2>(p, rows_total, tiles, di, st);
}

int launch_gg_fp4(const moe_gg_fp4_args* a, bool masked, void* stream) {
    if (!a) return fail(MOE_ERR_INVALID, "args is NULL");
    if (a->G <= 0 || a->N <= 0 || a->K <= 0 || a->M < 0)
        return fail(MOE_ERR_INVALID, "G, N, K must be positive and M non-negative (G=%d M=%d N=%d K=%d)", a->G, a->M, a->N, a->K);
    if (a->K % 128 != 0) return fail(MOE_ERR_INVALID, "K=%d must be a multiple of 128", a->K);
    if (a->N % 8 != 0) return fail(MOE_ERR_INVALID, "N=%d must be a multiple of 8", a->N);
    if (a->format != MOE_FP4_NV && a->format != MOE_FP4_MX) return fail(MOE_ERR_INVALID, "format must be MOE_FP4_NV or MOE_FP4_MX");
    if (a->d_dtype != MOE_DTYPE_BF16 && a->d_dtype != MOE_DTYPE_F32) return fail(MOE_ERR_INVALID, "d_dtype must be MOE_DTYPE_BF16 or MOE_DTYPE_F32");
    if (a->ldd < a->N || a->ldd % 8 != 0) return fail(MOE_ERR_INVALID, "ldd=%lld must be >= N and a multiple of 8", (long long)a->ldd);
    if (masked && a->G > gg::MAX_MASKED_GROUPS) return fail(MOE_ERR_INVALID, "masked layout supports at most %d groups", gg::MAX_MASKED_GROUPS);
    const long long rows_total = masked ? (long long)a->G * a->M : (long long)a->M;
    if (rows_total > 0x7FFFFFFFll || (long long)a->G * a->N > 0x7FFFFFFFll) return fail(MOE_ERR_INVALID, "row counts exceed 2^31-1");
    const long long chunks = (masked ? (long long)a->G : 1) * ((a->M + 127ll) / 128) + (long long)a->G * ((a->N + 127ll) / 128);
    if (chunks * ((a->K + 255ll) / 256) > 0x7FFFFFFFll / 256) return fail(MOE_ERR_INVALID, "the scales exceed 2^31 64-bit words");
    if (a->alpha && a->alpha_stride != 0 && a->alpha_stride != 1) return fail(MOE_ERR_INVALID, "alpha_stride must be 0 or 1");
    if (rows_total == 0) return MOE_OK;
    if (!a->a || !a->sfa || !a->b || !a->sfb || !a->layout || !a->d) return fail(MOE_ERR_INVALID, "a, sfa, b, sfb, layout and d must all be non-NULL");
    if (!aligned16(a->a) || !aligned16(a->sfa) || !aligned16(a->b) || !aligned16(a->sfb) || !aligned16(a->d))
        return fail(MOE_ERR_INVALID, "a, sfa, b, sfb and d must be 16-byte aligned");
    DeviceInfo* di = nullptr;
    int rc = device_info(&di);
    if (rc != MOE_OK) return rc;
    GGFp4Params p = {};
    p.a = static_cast<const uint8_t*>(a->a); p.b = static_cast<const uint8_t*>(a->b);
    p.sfa = static_cast<const uint8_t*>(a->sfa); p.sfb = static_cast<const uint8_t*>(a->sfb);
    p.alpha = a->alpha; p.alpha_stride = a->alpha_stride;
    p.layout = a->layout; p.rows_used = masked ? nullptr : a->rows_used;
    p.d = a->d; p.ldd = a->ldd; p.d_f32 = a->d_dtype == MOE_DTYPE_F32;
    p.G = a->G; p.M = a->M; p.N = a->N; p.K = a->K; p.masked = masked;
    p.kt = (a->K + 255) / 256 * (a->format == MOE_FP4_NV ? 4 : 2);
    p.a_tiles = (a->M + 127) / 128; p.b_tiles = (a->N + 127) / 128;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool nv = a->format == MOE_FP4_NV;
    if (a->M <= 32 && a->G <= (1 << 20)) return nv ? launch_fp4_few<true, 32>(p, rows_total, di, st) : launch_fp4_few<false, 32>(p, rows_total, di, st);
    // Tiles of 128 x 128 and one block each where one round of them covers the matrix: pairs of blocks on 256 x 256 would
    // leave most SMs idle (8 groups of 200 rows, 1024 x 1024: 7.3 us against 8.8; one of 256, 4096 x 7168: 13.1 against 15.3),
    // with more tiles they read less (one of 1024 rows, 4096 x 7168: 26 us against 19).
    const long long row_chunks = (a->M + 127) / 128 * (masked ? (long long)a->G : 1);
    const bool one_round = row_chunks * ((a->N + 127) / 128) <= di->num_sms && fp4_few_entries(p, 128) <= ff::LIST_CAP &&
                           (masked || a->M <= ff::MAX_ROWS) && a->G <= (1 << 20);
    if ((a->M <= 128 && a->G <= (1 << 20)) || one_round) return nv ? launch_fp4_few<true, 128>(p, rows_total, di, st) : launch_fp4_few<false, 128>(p, rows_total, di, st);
    return nv ? launch_fp4_pair_layout<true>(p, rows_total, di, st) : launch_fp4_pair_layout<false>(p, rows_total, di, st);
}

}  // namespace

extern "C" {

int moe_rms_norm_quant(const moe_norm_args* a, void* stream) {
    if (!a) return fail(MOE_ERR_INVALID, "args is NULL");
    int rc = check_norm(a->T, a->H, a->dtype, a->w_dtype);
    if (rc != MOE_OK || a->T == 0) return rc;
    if ((rc = check_rows("x", a->x, a->x_stride, a->H)) != MOE_OK) return rc;
    if (a->residual && (rc = check_rows("residual", a->residual, a->residual_stride, a->H)) != MOE_OK) return rc;
    if (!a->weight || !a->q || !a->scales || !a->rstd || (a->residual && !a->h))
        return fail(MOE_ERR_INVALID, "weight, q, scales, rstd (and h, with a residual) must be non-NULL");
    if (!aligned16(a->weight) || !aligned16(a->q) || !aligned16(a->h) || !aligned16(a->y))
        return fail(MOE_ERR_INVALID, "weight, q, h and y must be 16-byte aligned");
    DeviceInfo* di = nullptr;
    if ((rc = device_info(&di)) != MOE_OK) return rc;
    NormParams p = {};
    p.x = a->x; p.x_stride = a->x_stride; p.residual = a->residual; p.res_stride = a->residual_stride;
    p.weight = a->weight; p.q = static_cast<uint8_t*>(a->q); p.scales = a->scales; p.ss_row = a->ss_row; p.ss_blk = a->ss_blk;
    p.h = a->h; p.y = a->y; p.rstd = a->rstd; p.T = a->T; p.H = a->H; p.eps = a->eps; p.pow2 = a->pow2 ? 1 : 0;
    const NormShape s = norm_shape(a->H);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        rc = a->w_dtype == a->dtype ? launch_norm<T, T>(p, s, di, st) : launch_norm<T, float>(p, s, di, st);
    });
    return rc;
}

size_t moe_rms_norm_backward_workspace_bytes(int32_t T, int32_t H) {
    if (T < 0 || H <= 0 || H > NORM_MAX_H) return 0;
    const int parts = norm_grad_parts(H);
    return align256((size_t)(T < parts ? (T > 0 ? T : 1) : parts) * (size_t)H * 4);
}

int moe_rms_norm_backward(const moe_norm_grad_args* a, void* stream) {
    if (!a) return fail(MOE_ERR_INVALID, "args is NULL");
    int rc = check_norm(a->T, a->H, a->dtype, a->w_dtype);
    if (rc != MOE_OK) return rc;
    if (!a->dw || !aligned16(a->dw)) return fail(MOE_ERR_INVALID, "dw must be non-NULL and 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->T == 0) {
        CUDA_TRY(cudaMemsetAsync(a->dw, 0, (size_t)a->H * 4, st));
        return MOE_OK;
    }
    if ((rc = check_rows("dy", a->dy, a->dy_stride, a->H)) != MOE_OK) return rc;
    if ((rc = check_rows("h", a->h, a->h_stride, a->H)) != MOE_OK) return rc;
    if (a->dh && (rc = check_rows("dh", a->dh, a->dh_stride, a->H)) != MOE_OK) return rc;
    if (!a->weight || !a->rstd || !a->dx || !aligned16(a->weight) || !aligned16(a->dx))
        return fail(MOE_ERR_INVALID, "weight, rstd and dx must be non-NULL, weight and dx 16-byte aligned");
    if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < moe_rms_norm_backward_workspace_bytes(a->T, a->H))
        return fail(MOE_ERR_INVALID, "workspace too small or not 16-byte aligned (moe_rms_norm_backward_workspace_bytes)");
    DeviceInfo* di = nullptr;
    if ((rc = device_info(&di)) != MOE_OK) return rc;
    NormGradParams p = {};
    p.dy = a->dy; p.dy_stride = a->dy_stride; p.h = a->h; p.h_stride = a->h_stride; p.weight = a->weight; p.rstd = a->rstd;
    p.dh = a->dh; p.dh_stride = a->dh_stride; p.dx = a->dx; p.partial = static_cast<float*>(a->workspace); p.T = a->T; p.H = a->H;
    const NormShape s = norm_shape(a->H);
    with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        rc = a->w_dtype == a->dtype ? launch_norm_grad<T, T>(p, a->dw, s, di, st) : launch_norm_grad<T, float>(p, a->dw, s, di, st);
    });
    return rc;
}

int moe_route(const moe_route_args* a, void* stream) {
    if (!a) return fail(MOE_ERR_INVALID, "args is NULL");
    int rc = check_route(a->T, a->E, a->top_k, a->dtype, a->score, a->stride);
    if (rc != MOE_OK) return rc;
    if (a->n_group <= 0 || a->n_group > RT_MAX_GROUPS || a->E % a->n_group)
        return fail(MOE_ERR_INVALID, "n_group=%d must be in [1, %d] and divide E=%d", a->n_group, RT_MAX_GROUPS, a->E);
    if (a->topk_group <= 0 || a->topk_group > a->n_group) return fail(MOE_ERR_INVALID, "topk_group must be in [1, n_group]");
    if ((int64_t)a->topk_group * (a->E / a->n_group) < a->top_k) return fail(MOE_ERR_INVALID, "the kept groups hold fewer than top_k=%d experts", a->top_k);
    if (a->group_score != MOE_GROUP_MAX && a->group_score != MOE_GROUP_TOP2) return fail(MOE_ERR_INVALID, "group_score must be MOE_GROUP_MAX or MOE_GROUP_TOP2");
    if (a->bias && a->bias_dtype != MOE_DTYPE_BF16 && a->bias_dtype != MOE_DTYPE_F32) return fail(MOE_ERR_INVALID, "bias_dtype must be bf16 or f32");
    if (a->T == 0) return MOE_OK;
    if (!a->logits || !a->ids || !a->weights) return fail(MOE_ERR_INVALID, "logits, ids and weights must be non-NULL");
    RouteParams p;
    p.logits = a->logits; p.stride = a->stride; p.bias = a->bias; p.bias_bf16 = a->bias_dtype == MOE_DTYPE_BF16;
    p.ids = a->ids; p.weights = a->weights; p.T = a->T; p.E = a->E; p.top_k = a->top_k; p.n_group = a->n_group;
    p.topk_group = a->topk_group; p.sigmoid = a->score == MOE_SCORE_SIGMOID; p.top2 = a->group_score == MOE_GROUP_TOP2;
    p.renorm = a->renormalize ? 1 : 0; p.vec = route_vec(a->logits, a->stride, a->E, a->dtype); p.scale = a->scale;
    p.bias_vec = route_vec(a->bias, 0, a->E, a->bias_dtype);
    p.gs = a->E / a->n_group;
    const int per = route_per_lane(a->E), lanes = p.gs / per;
    p.group_shift = lanes * per == p.gs && lanes > 0 && (lanes & (lanes - 1)) == 0 ? __builtin_ctz(lanes) : -1;
    const size_t smem = a->bias || a->n_group > 1 ? (size_t)RT_WARPS * a->E * 8 : 0;
    with_dtype(a->dtype, [&](auto t) { launch_route<decltype(t)>(p, smem, static_cast<cudaStream_t>(stream)); });
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

int moe_route_backward(const moe_route_grad_args* a, void* stream) {
    if (!a) return fail(MOE_ERR_INVALID, "args is NULL");
    int rc = check_route(a->T, a->E, a->top_k, a->dtype, a->score, a->stride);
    if (rc != MOE_OK || a->T == 0) return rc;
    if (!a->grad_weights || !a->logits || !a->ids || !a->dlogits) return fail(MOE_ERR_INVALID, "grad_weights, logits, ids and dlogits must be non-NULL");
    RouteGradParams p;
    p.grad = a->grad_weights; p.logits = a->logits; p.stride = a->stride; p.ids = a->ids; p.out = a->dlogits;
    p.T = a->T; p.E = a->E; p.top_k = a->top_k; p.sigmoid = a->score == MOE_SCORE_SIGMOID; p.renorm = a->renormalize ? 1 : 0;
    p.vec = route_vec(a->logits, a->stride, a->E, a->dtype) && aligned16(a->dlogits); p.scale = a->scale;
    with_dtype(a->dtype, [&](auto t) { launch_route_grad<decltype(t)>(p, static_cast<cudaStream_t>(stream)); });
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

size_t moe_quant_fp4_workspace_bytes(int32_t rows, int32_t src_rows, int32_t K, int32_t format) {
    if (src_rows <= 0 || K <= 0 || K % 128 || rows < 2ll * src_rows || (long long)rows * K < FP4_COPY_FROM || (format != MOE_FP4_NV && format != MOE_FP4_MX)) return 0;
    return align256((size_t)src_rows * (size_t)(K / 2)) + align256((size_t)src_rows * ((K + 255ll) / 256) * (format == MOE_FP4_NV ? 16 : 8));
}

int moe_quant_fp4(const moe_fp4_quant_args* a, void* stream) {
    if (!a) return fail(MOE_ERR_INVALID, "args is NULL");
    if (a->groups <= 0 || a->groups > 65535 || a->rows < 0 || a->rows > MAX_ROWS_32 || a->src_rows < 0 || a->K <= 0 || a->K % 128)
        return fail(MOE_ERR_INVALID, "groups must be in [1, 65535], rows=%d in [0, %d] and K=%d a positive multiple of 128", a->rows, MAX_ROWS_32, a->K);
    if (a->format != MOE_FP4_NV && a->format != MOE_FP4_MX) return fail(MOE_ERR_INVALID, "format must be MOE_FP4_NV or MOE_FP4_MX");
    if (!float_dtype(a->dtype)) return fail(MOE_ERR_INVALID, "dtype must be bf16, f16 or f32");
    if (a->src_pair ? a->groups != 1 || a->top_k <= 0 : a->rows != a->src_rows)
        return fail(MOE_ERR_INVALID, "src_pair needs one group and a positive top_k; without it rows and src_rows are the same");
    if (a->factor && a->format == MOE_FP4_MX) return fail(MOE_ERR_INVALID, "mxfp4 has no factor");
    if (a->rows == 0) return MOE_OK;
    if (!a->q || !a->scales || (!a->x && a->src_rows > 0)) return fail(MOE_ERR_INVALID, "x, q and scales must be non-NULL");
    const int64_t cols = a->silu_mul ? 2ll * a->K : a->K;
    if (!aligned16(a->x) || a->x_stride < cols || a->x_stride % 8) return fail(MOE_ERR_INVALID, "x must be 16-byte aligned with a row stride that covers its columns and is a multiple of 8");
    if (!aligned16(a->q) || !aligned16(a->scales)) return fail(MOE_ERR_INVALID, "q and scales must be 16-byte aligned");
    Fp4QuantParams p = {};
    p.x = a->x; p.x_stride = a->x_stride; p.factor = a->factor; p.factor_stride = a->factor_stride; p.src = a->src_pair; p.top_k = a->top_k;
    p.q = static_cast<uint8_t*>(a->q); p.sf = static_cast<uint8_t*>(a->scales); p.rows = a->rows; p.K = a->K;
    p.gate_first = a->gate_first ? 1 : 0; p.src_rows = a->src_rows; p.k_blocks = (a->K + 255) / 256;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t need = a->src_pair && !a->silu_mul ? moe_quant_fp4_workspace_bytes(a->rows, a->src_rows, a->K, a->format) : 0;
    const bool copy = need > 0 && a->workspace != nullptr;
    if (copy) {
        if (!aligned16(a->workspace) || a->workspace_bytes < need) return fail(MOE_ERR_INVALID, "workspace too small or not 16-byte aligned (moe_quant_fp4_workspace_bytes)");
        p.src = nullptr; p.rows = a->src_rows; p.q = static_cast<uint8_t*>(a->workspace); p.sf = p.q + align256((size_t)a->src_rows * (size_t)(a->K / 2));
    }
    const auto row_pieces = [](int rows) { return (long long)((rows + 127ll) / 128) * (128 / FP4_QUANT_ROWS); };
    if (row_pieces(a->rows) * p.k_blocks > 0x7FFFFFFFll) return fail(MOE_ERR_INVALID, "rows x K exceeds what one call covers");
    const dim3 grid((unsigned)(row_pieces(p.rows) * p.k_blocks), a->groups, 1);
    with_dtype(a->dtype, [&](auto t) { launch_quant_fp4<decltype(t)>(p, a->format == MOE_FP4_NV, a->silu_mul != 0, copy, grid, st); });
    CUDA_TRY(cudaGetLastError());
    if (copy) {
        const Fp4CopyParams c = {p.q, reinterpret_cast<const uint32_t*>(p.sf), a->src_pair, a->top_k, static_cast<uint8_t*>(a->q), static_cast<uint32_t*>(a->scales),
                                 a->rows, a->src_rows, a->K, p.k_blocks, (a->K + FP4_COPY_COLS - 1) / FP4_COPY_COLS};
        CUDA_TRY(launch_pdl(a->format == MOE_FP4_NV ? copy_fp4_rows_kernel<true> : copy_fp4_rows_kernel<false>, dim3((unsigned)(row_pieces(a->rows) * c.pieces)),
                            dim3(FP4_QUANT_THREADS), 0, st, c));
    }
    return MOE_OK;
}

int moe_unpack_fp4(const void* q, void* out_e4m3, int64_t n_bytes, void* stream) {
    if (n_bytes < 0 || n_bytes % 8) return fail(MOE_ERR_INVALID, "n_bytes must be a non-negative multiple of 8");
    if (n_bytes == 0) return MOE_OK;
    if (!q || !out_e4m3 || !aligned16(q) || !aligned16(out_e4m3)) return fail(MOE_ERR_INVALID, "q and out must be non-NULL and 16-byte aligned");
    constexpr int each = FP4_UNPACK_THREADS * FP4_UNPACK_EACH;
    const long long n = n_bytes / 8, blocks = (n + each - 1) / each;
    if (blocks > 0x7FFFFFFFll) return fail(MOE_ERR_INVALID, "n_bytes exceeds what one call covers");
    unpack_fp4_kernel<<<(unsigned)blocks, FP4_UNPACK_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const uint2*>(q), static_cast<uint4*>(out_e4m3), n);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

int moe_gg_fp4_contiguous(const moe_gg_fp4_args* args, void* stream) { return launch_gg_fp4(args, false, stream); }
int moe_gg_fp4_masked(const moe_gg_fp4_args* args, void* stream) { return launch_gg_fp4(args, true, stream); }

}  // extern "C"
