// GEMM dispatch: tensor maps, kernel-variant selection, launches, split-K reduce, the kernarg-blob drop-in
// and the on-device tuner.  Replaces the reference's kernel cache + AQL dispatch
// (GpuRuntime::ensure_kernel_t0 / dispatch, src/ignis/gpu_context.rs:171-288) and the Ignis GEMM entry
// points (src/ignis/ops/bf16_matmul.rs:162-308).
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "gemm_launch.cuh"
#include "t0b_internal.hpp"

using namespace t0b;

static constexpr int kTraceCtas = 160;   // CTAs per launch the timeline buffer has room for (T0B_TRACE_CTAS in the header)

namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver entry point is looked up at run time so the library links against the CUDA runtime only and
// can be loaded (for symbol checks) on a machine without a GPU driver.
EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// 2-D tensor map (bf16, or f32 when elem == 4): inner (contiguous) extent d0, outer extent d1, outer pitch ld
// elements, box b0 x b1, swizzled; out-of-bounds elements read as zero and are not written.
int32_t get_tmap(t0b_ctx* ctx, uint64_t ptr, uint64_t d0, uint64_t d1, uint64_t ld, uint32_t b0, uint32_t b1,
                 CUtensorMap* out, uint32_t elem = 2) {
    t0b_ctx::TmapKey key{ptr, d0, d1, ld, b0, b1, elem};
    auto it = ctx->tmaps.find(key);
    if (it != ctx->tmaps.end()) {
        *out = it->second;
        return T0B_OK;
    }
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return set_error(ctx, T0B_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[2] = {d0, d1};
    cuuint64_t strides[1] = {ld * elem};
    cuuint32_t box[2] = {b0, b1};
    cuuint32_t estr[2] = {1, 1};
    // Boxes with 128-byte rows (the operand tiles) use the 128-byte swizzle, boxes with 64-byte rows (the epilogue's
    // half tiles) the 64-byte swizzle.
    const CUtensorMapSwizzle swz = (b0 * elem == 64) ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    CUresult r = fn(out, elem == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, reinterpret_cast<void*>(ptr), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(ctx, T0B_ERR_INVALID,
                         "cuTensorMapEncodeTiled failed (%d) for ptr=%llx dims=(%llu,%llu) ld=%llu box=(%u,%u)",
                         static_cast<int>(r), static_cast<unsigned long long>(ptr), static_cast<unsigned long long>(d0),
                         static_cast<unsigned long long>(d1), static_cast<unsigned long long>(ld), b0, b1);
    if (ctx->tmaps.size() > 8192) ctx->tmaps.clear();
    ctx->tmaps.emplace(key, *out);
    return T0B_OK;
}

struct GemmCall {
    const t0b_gemm_config* cfg;
    int trans_a, trans_b;
    uint64_t a, b;
    uint64_t c_dst[kMaxDst];
    int n_dst;
    uint32_t m, n, k;
    uint64_t lda, ldb, ldc;
    int out_bf16;
    EpiChain epi;
    uint64_t workspace;
    size_t workspace_bytes;
    bool slabs_only;        // leave unreduced split-K slabs in c_dst[0] (reference contract)
    uint32_t force_split;   // for slabs_only: the exact number of slabs the caller expects
    bool no_auto_split;     // an automatically chosen config keeps the whole contraction in one tile (fixed summation order)
    bool accumulate;        // C += A*B (f32 output, one destination, never split)
    const int* dyn_rows;    // rows counted on the device (GemmParams)
    int dyn_off, dyn_k;
    bool late_wait;
};

// Expand the public single-op epilogue code into a chain (EPI_BIAS_RELU = bias add, then ReLU).
int32_t make_chain(t0b_ctx* ctx, const int32_t* ops, int n_ops, uint64_t bias, float alpha, float lo, float hi, EpiChain* out) {
    EpiChain e{};
    e.alpha = alpha; e.clamp_lo = lo; e.clamp_hi = hi; e.bias = reinterpret_cast<const float*>(bias);
    for (int i = 0; i < n_ops; ++i) {
        const int op = ops[i];
        if (op == EPI_STORE) continue;
        if (op < 0 || op > EPI_CLAMP) return set_error(ctx, T0B_ERR_INVALID, "gemm: unknown epilogue %d", op);
        const int expanded[2] = {op == EPI_BIAS_RELU ? EPI_BIAS : op, EPI_RELU};
        const int count = op == EPI_BIAS_RELU ? 2 : 1;
        for (int j = 0; j < count; ++j) {
            if (e.n >= kMaxEpiOps) return set_error(ctx, T0B_ERR_INVALID, "gemm: epilogue chain longer than %d operations", kMaxEpiOps);
            e.ops[e.n++] = expanded[j];
        }
        if ((op == EPI_BIAS || op == EPI_BIAS_RELU) && !bias)
            return set_error(ctx, T0B_ERR_INVALID, "gemm: bias epilogue without a bias pointer");
    }
    *out = e;
    return T0B_OK;
}

uint64_t slab_pitch(uint64_t n) { return (n + 3) & ~3ull; }

int32_t launch_reduce(t0b_ctx* ctx, const float* partial, uint32_t sk, uint32_t m, uint32_t n, uint64_t slab_stride,
                      uint64_t ld_partial, bool padded, void* c, uint64_t ldc, int out_bf16, const EpiChain& epi) {
    ReduceParams rp{partial, static_cast<long long>(slab_stride), static_cast<long long>(ld_partial), c,
                    static_cast<long long>(ldc), epi, static_cast<int>(m), static_cast<int>(n),
                    static_cast<int>(sk), out_bf16, padded ? 1 : 0};
    const long long total = static_cast<long long>(m) * ((n + 3) / 4);
    const int blocks = static_cast<int>(std::min<long long>((total + 255) / 256, static_cast<long long>(ctx->num_sms) * 8));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::max(blocks, 1));
    cfg.blockDim = dim3(256);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // scheduled as the GEMM's CTAs exit
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    cudaLaunchKernelEx(&cfg, splitk_reduce_kernel, rp);
    return check_cuda(ctx, cudaGetLastError(), "splitk_reduce launch");
}

// The config a call runs: its own, else a forced preset (T0_FORCE_CONFIG), else measured in this process (t0b_tune), else
// the table shipped with the library, else the cost model.
int32_t choose_config(t0b_ctx* ctx, const GemmCall& g, t0b_gemm_config* cfg, const char** source) {
    if (g.cfg) {
        *cfg = *g.cfg;
        return T0B_OK;
    }
    int tuned_source = 0;
    if (!ctx->force_config.empty()) {
        if (t0b_config_preset(ctx->force_config.c_str(), cfg) != T0B_OK)
            return set_error(ctx, T0B_ERR_INVALID, "gemm: T0_FORCE_CONFIG=%s is not a preset name", ctx->force_config.c_str());
        *source = "forced";
    } else if (tuned_lookup(g.m, g.n, g.k, g.trans_a, g.trans_b, g.out_bf16, cfg, &tuned_source)) {
        *source = tuned_source == 2 ? "tuned in this process" : "shipped table";
    } else {
        default_b200_config(g.m, g.k, g.n, ctx->num_sms, cfg);
        *source = "cost model";
    }
    if (g.no_auto_split) cfg->split_k = 0;
    return T0B_OK;
}

// Whether the split-K of this plan runs inside thread-block clusters (no slabs in global memory).
bool splitk_in_cluster(t0b_ctx* ctx, const GemmCall& g, const t0b_gemm_plan& plan) {
    if (g.slabs_only || plan.split_k <= 1 || plan.split_k > 8 || (plan.split_k & (plan.split_k - 1)) != 0 || g.n_dst != 1 || !plan.use_tma ||
        plan.cta_group != 1 || plan.m_tiles != 1 || plan.n_tiles != 1 || !ctx->cluster_splitk)
        return false;
    if (plan.split_k > 4) {
        // Eight-CTA clusters do not tile every GPC: when the tiles need more clusters than fit at once, the second wave
        // costs more than the slab round trip saves.
        const int tiles = static_cast<int>(((g.m + plan.bm - 1) / plan.bm) * ((g.n + plan.bn - 1) / plan.bn));
        const int fit = plan.bn == 256 ? max_active_splitk_clusters<256>(ctx, plan.split_k)
                                       : (plan.bn == 128 ? max_active_splitk_clusters<128>(ctx, plan.split_k)
                                                         : max_active_splitk_clusters<64>(ctx, plan.split_k));
        if (tiles > fit) return false;
    }
    return true;
}

// Rasterisation group width: concurrently running tiles should cover a square-ish patch of C, so that A and B panels are
// shared through L2: group * bm ~= (clusters / group) * bn.
int raster_group(t0b_ctx* ctx, uint32_t bm, uint32_t bn, uint32_t cta_group, bool swap_grid) {
    const double clusters = static_cast<double>(ctx->num_sms) / cta_group;
    const int grp = static_cast<int>(std::lround(std::sqrt(clusters * (swap_grid ? bn : bm) / static_cast<double>(swap_grid ? bm : bn))));
    return std::max(1, std::min(grp, 16));
}

// The kernel of a plan's tile.
template <int KIND>
int32_t launch_plan(t0b_ctx* ctx, const t0b_gemm_plan& plan, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                    const KernelParams<KIND>& p, int num_work) {
    if (plan.cta_group == 2) {
        if (plan.n_tiles == 2) return launch_variant<256, 2, 2, 1, KIND>(ctx, ta, tb, tc, p, num_work);
        if (plan.m_tiles == 2) return launch_variant<256, 2, 2, 0, KIND>(ctx, ta, tb, tc, p, num_work);
        if (plan.bn == 256) return launch_variant<256, 2, 1, 0, KIND>(ctx, ta, tb, tc, p, num_work);
        return launch_variant<128, 2, 1, 0, KIND>(ctx, ta, tb, tc, p, num_work);
    }
    if (plan.bn == 256) return launch_variant<256, 1, 1, 0, KIND>(ctx, ta, tb, tc, p, num_work, p.cluster_sk);
    if (plan.bn == 128) return launch_variant<128, 1, 1, 0, KIND>(ctx, ta, tb, tc, p, num_work, p.cluster_sk);
    return launch_variant<64, 1, 1, 0, KIND>(ctx, ta, tb, tc, p, num_work, p.cluster_sk);
}

int32_t run_gemm(t0b_ctx* ctx, const GemmCall& g) {
    if (g.m == 0 || g.n == 0) return T0B_OK;
    if (!g.a || !g.b || g.n_dst < 1 || g.n_dst > kMaxDst)
        return set_error(ctx, T0B_ERR_INVALID, "gemm: null operand or bad destination count");
    for (int d = 0; d < g.n_dst; ++d)
        if (!g.c_dst[d]) return set_error(ctx, T0B_ERR_INVALID, "gemm: null destination %d", d);
    const uint64_t min_lda = g.trans_a ? g.m : g.k, min_ldb = g.trans_b ? g.k : g.n;
    if (g.lda < min_lda || g.ldb < min_ldb || g.ldc < g.n)
        return set_error(ctx, T0B_ERR_INVALID, "gemm: leading dimension smaller than the row length (lda=%llu ldb=%llu ldc=%llu)",
                         static_cast<unsigned long long>(g.lda), static_cast<unsigned long long>(g.ldb),
                         static_cast<unsigned long long>(g.ldc));

    {
        // An operand that starts one of this runtime's own allocations must fit in it: an undersized buffer is reported
        // here instead of faulting on the device.  (Pointers from elsewhere, or into the middle of a buffer, are not known.)
        std::lock_guard<std::recursive_mutex> lk(ctx->mu);
        auto too_small = [&](uint64_t ptr, uint64_t rows, uint64_t cols, uint64_t ld, size_t elem_bytes, uint64_t* have) {
            auto it = ctx->live.find(reinterpret_cast<void*>(ptr));
            if (it == ctx->live.end() || rows == 0 || cols == 0) return false;
            *have = it->second;
            return ((rows - 1) * ld + cols) * elem_bytes > it->second;
        };
        uint64_t have = 0;
        if (too_small(g.a, g.trans_a ? g.k : g.m, g.trans_a ? g.m : g.k, g.lda, 2, &have))
            return set_error(ctx, T0B_ERR_INVALID, "gemm: A (%u x %u bf16) does not fit its %llu-byte buffer", g.m, g.k,
                             static_cast<unsigned long long>(have));
        if (too_small(g.b, g.trans_b ? g.n : g.k, g.trans_b ? g.k : g.n, g.ldb, 2, &have))
            return set_error(ctx, T0B_ERR_INVALID, "gemm: B (%u x %u bf16) does not fit its %llu-byte buffer", g.k, g.n,
                             static_cast<unsigned long long>(have));
        if (!g.slabs_only)
            for (int d = 0; d < g.n_dst; ++d)
                if (too_small(g.c_dst[d], g.m, g.n, g.ldc, g.out_bf16 ? 2 : 4, &have))
                    return set_error(ctx, T0B_ERR_INVALID, "gemm: C (%u x %u) does not fit its %llu-byte buffer", g.m, g.n,
                                     static_cast<unsigned long long>(have));
    }

    t0b_gemm_config cfg;
    const char* cfg_source = "caller";
    int32_t rc_cfg = choose_config(ctx, g, &cfg, &cfg_source);
    if (rc_cfg != T0B_OK) return rc_cfg;
    if (g.slabs_only) cfg.split_k = g.force_split;
    if (g.accumulate) cfg.split_k = 0;
    if (cfg.split_k > 1 && (cfg.split_k & (cfg.split_k - 1)) != 0)
        return set_error(ctx, T0B_ERR_INVALID, "gemm: split_k=%u must be a power of 2", cfg.split_k);

    t0b_gemm_plan plan;
    PlanInput pin{g.m, g.n, g.k, g.trans_a, g.trans_b, g.lda, g.ldb, g.a, g.b, ctx->num_sms};
    resolve_plan(&cfg, pin, &plan);

    if (ctx->dump_config) {
        // One line per new (shape, layout, output, config) on stderr: what was chosen, by whom, and what it runs as.
        char name[96], line[320];
        t0b_config_name(&cfg, name, sizeof(name));
        std::snprintf(line, sizeof(line), "t0b gemm %ux%ux%u %c%c %s dst=%d: %s (%s) -> tile %ux%u cta_group %u stages %u split_k %u%s",
                      g.m, g.n, g.k, g.trans_a ? 'T' : 'N', g.trans_b ? 'T' : 'N', g.out_bf16 ? "bf16" : "f32", g.n_dst, name, cfg_source,
                      plan.bm, plan.bn, plan.cta_group, plan.stages, plan.split_k, plan.use_tma ? "" : " (CUDA-core kernel)");
        if (ctx->dumped.emplace(line, 1).second) std::fprintf(stderr, "%s\n", line);
    }
    if (g.accumulate && (g.out_bf16 || g.n_dst != 1 || g.slabs_only || !plan.use_tma))
        return set_error(ctx, T0B_ERR_INVALID, "gemm: accumulation needs one f32 destination and operands TMA can address");
    const size_t elem = g.out_bf16 ? 2 : 4;
    if (g.k == 0) {
        if (g.accumulate) return T0B_OK;
        // Empty contraction: every accumulator is +0.0, so the result is epilogue(0).
        if (g.slabs_only) {
            // Every slab the caller expects carries an empty K range (the slabs are dense and adjacent).
            return check_cuda(ctx, cudaMemsetAsync(reinterpret_cast<void*>(g.c_dst[0]), 0,
                                                   static_cast<size_t>(g.force_split) * g.m * g.n * 4, ctx->stream),
                              "cudaMemsetAsync(k=0 slabs)");
        }
        for (int d = 0; d < g.n_dst; ++d) {
            if (g.epi.n == 0) {
                int32_t rc = check_cuda(ctx, cudaMemset2DAsync(reinterpret_cast<void*>(g.c_dst[d]), g.ldc * elem, 0, g.n * elem, g.m,
                                                               ctx->stream), "cudaMemset2DAsync(k=0)");
                if (rc != T0B_OK) return rc;
                continue;
            }
            // With a fused store-phase chain the CUDA-core kernel applies it to the zero accumulators.
            SimtParams sp{};
            sp.a = reinterpret_cast<const __nv_bfloat16*>(g.a);
            sp.b = reinterpret_cast<const __nv_bfloat16*>(g.b);
            sp.lda = g.lda; sp.ldb = g.ldb; sp.M = g.m; sp.N = g.n; sp.K = 0;
            sp.trans_a = g.trans_a; sp.trans_b = g.trans_b; sp.k_begin = 0; sp.k_end = 0;
            sp.c = reinterpret_cast<void*>(g.c_dst[d]); sp.ldc = g.ldc; sp.out_bf16 = g.out_bf16; sp.epi = g.epi;
            dim3 grid((g.n + 63) / 64, (g.m + 63) / 64);
            gemm_bf16_simt_kernel<<<grid, 256, 0, ctx->stream>>>(sp);
            int32_t rc = check_cuda(ctx, cudaGetLastError(), "simt gemm launch (k=0)");
            if (rc != T0B_OK) return rc;
            ++ctx->launches;
        }
        return T0B_OK;
    }

    // Split-K inside clusters (see below) needs no slabs at all.
    const bool cluster_sk_possible = splitk_in_cluster(ctx, g, plan);
    // Where do split-K partials go?
    float* partial = nullptr;
    uint64_t slab_stride = static_cast<uint64_t>(g.m) * g.n, ld_partial = g.n;
    uint32_t sk = plan.split_k;
    // Slabs of its own a call lays out at a pitch of whole 16 bytes, which the sum reads and the epilogue writes in float4; a caller's
    // workspace may have been sized for the plain pitch.
    const uint64_t pitch4 = slab_pitch(g.n);
    if (!g.slabs_only && (!g.workspace || g.workspace_bytes >= static_cast<uint64_t>(sk) * g.m * pitch4 * 4)) {
        ld_partial = pitch4;
        slab_stride = static_cast<uint64_t>(g.m) * pitch4;
    }
    if (g.slabs_only) {
        partial = reinterpret_cast<float*>(g.c_dst[0]);
        if (sk < g.force_split) {
            // K has fewer 64-blocks than slabs were asked for: the trailing slabs carry no K range.
            int32_t rc = check_cuda(ctx, cudaMemsetAsync(partial + slab_stride * sk, 0,
                                                         slab_stride * 4 * (g.force_split - sk), ctx->stream),
                                    "cudaMemsetAsync(empty slabs)");
            if (rc != T0B_OK) return rc;
        }
    } else if (sk > 1 && !cluster_sk_possible) {
        const size_t need = static_cast<size_t>(sk) * slab_stride * 4;
        if (g.workspace) {
            if (g.workspace_bytes < need)
                return set_error(ctx, T0B_ERR_INVALID, "gemm: split-K workspace too small (%zu < %zu bytes)",
                                 g.workspace_bytes, need);
            partial = reinterpret_cast<float*>(g.workspace);
        } else {
            if (ctx->ws_bytes < need) {
                if (ctx->capturing) return set_error(ctx, T0B_ERR_INVALID, "gemm: cannot grow the workspace during graph capture");
                cudaStreamSynchronize(ctx->stream);
                if (ctx->ws) cudaFree(ctx->ws);
                ctx->ws = nullptr;
                ctx->ws_bytes = 0;
                int32_t rc = check_cuda(ctx, cudaMalloc(&ctx->ws, need), "cudaMalloc(workspace)");
                if (rc != T0B_OK) return rc;
                ctx->ws_bytes = need;
            }
            partial = static_cast<float*>(ctx->ws);
        }
    }
    const bool to_slabs = g.slabs_only || sk > 1;
    // Split-K on a single-CTA tile with up to eight K ranges runs as thread-block clusters: the CTAs of a cluster take the
    // K ranges of one tile, keep their partial tiles in shared memory and sum them over distributed shared memory in
    // K-range order -- one launch, no slabs in global memory, the same bits as the slab sum.  T0B_CLUSTER_SPLITK=0 keeps
    // the slab path (GEMM into slabs + reduce kernel), as do CTA-pair tiles, more than eight ranges, the unreduced-slab
    // contract and operands TMA cannot address.
    const bool cluster_sk = cluster_sk_possible;

    if (!plan.use_tma) {
        // Operands TMA cannot address: CUDA-core kernel, one launch per K range.
        for (uint32_t s = 0; s < sk; ++s) {
            SimtParams sp{};
            sp.a = reinterpret_cast<const __nv_bfloat16*>(g.a);
            sp.b = reinterpret_cast<const __nv_bfloat16*>(g.b);
            sp.lda = g.lda; sp.ldb = g.ldb;
            sp.M = g.m; sp.N = g.n; sp.K = g.k;
            sp.trans_a = g.trans_a; sp.trans_b = g.trans_b;
            sp.k_begin = static_cast<int>(std::min<uint64_t>(g.k, static_cast<uint64_t>(s) * plan.kb_per_split * 64));
            sp.k_end = static_cast<int>(std::min<uint64_t>(g.k, static_cast<uint64_t>(s + 1) * plan.kb_per_split * 64));
            const int ndst = to_slabs ? 1 : g.n_dst;
            for (int d = 0; d < ndst; ++d) {
                if (to_slabs) {
                    sp.c = partial + slab_stride * s; sp.ldc = ld_partial; sp.out_bf16 = 0; sp.epi = EpiChain{};
                } else {
                    sp.c = reinterpret_cast<void*>(g.c_dst[d]); sp.ldc = g.ldc; sp.out_bf16 = g.out_bf16; sp.epi = g.epi;
                }
                dim3 grid((g.n + 63) / 64, (g.m + 63) / 64);
                gemm_bf16_simt_kernel<<<grid, 256, 0, ctx->stream>>>(sp);
                int32_t rc = check_cuda(ctx, cudaGetLastError(), "simt gemm launch");
                if (rc != T0B_OK) return rc;
                ++ctx->launches;
            }
        }
    } else {
        CUtensorMap ta, tb;
        int32_t rc;
        if (!g.trans_a) rc = get_tmap(ctx, g.a, g.k, g.m, g.lda, 64, 128, &ta);
        else rc = get_tmap(ctx, g.a, g.m, g.k, g.lda, 64, 64, &ta);
        if (rc != T0B_OK) return rc;
        const uint32_t bn_cta = (plan.n_tiles == 2 ? 256u : plan.bn) / plan.cta_group;
        if (g.trans_b) rc = get_tmap(ctx, g.b, g.k, g.n, g.ldb, 64, bn_cta, &tb);
        else rc = get_tmap(ctx, g.b, g.n, g.k, g.ldb, 64, 64, &tb);
        if (rc != T0B_OK) return rc;

        KernelParams<0> p{};
        for (int d = 0; d < g.n_dst; ++d) p.c_dst[d] = reinterpret_cast<void*>(g.c_dst[d]);
        p.n_dst = g.n_dst;
        p.ldc = static_cast<long long>(g.ldc);
        p.epi = g.epi;
        p.partial = to_slabs ? partial : nullptr;
        p.slab_stride = static_cast<long long>(slab_stride);
        p.ld_partial = static_cast<long long>(ld_partial);
        p.M = g.m; p.N = g.n; p.K = g.k;
        p.tiles_m = (g.m + plan.bm - 1) / plan.bm;
        p.tiles_n = (g.n + plan.bn - 1) / plan.bn;
        // The kernel routes to the slab path when split_k > 1; a single requested slab is the plain store.
        p.split_k = static_cast<int>(sk);
        p.kb_total = (g.k + 63) / 64;
        p.kb_per_split = plan.kb_per_split;
        p.a_mn_major = g.trans_a ? 1 : 0;     // A stored [K,M]: M contiguous
        p.b_mn_major = g.trans_b ? 0 : 1;     // B stored [K,N]: N contiguous
        p.out_bf16 = g.out_bf16;
        p.raster_along_n = cfg.swap_grid ? 0 : 1;
        {
            p.group = raster_group(ctx, plan.bm, plan.bn, plan.cta_group, cfg.swap_grid != 0);
            // A measured group width travels in the config (lds_pad, the reference's RDNA3 padding knob, has no other
            // meaning here): the tuner tries a few and the shipped table keeps the winner -- on tall shapes the panel
            // order is worth up to a fifth of the run time.
            if (cfg.lds_pad > 0) p.group = static_cast<int>(std::min<uint32_t>(cfg.lds_pad, 4096u));
            if (ctx->raster_group > 0) p.group = ctx->raster_group;
        }
        p.mn_lbo = 8192; p.mn_sbo = 1024; p.mn_kstep = 2048;
        p.status = ctx->status_dev;
        p.wait_limit_ns = ctx->wait_limit_ns;
        p.wait_hint_ns = ctx->wait_hint_ns;
        if (g.slabs_only && sk == 1) {
            // One slab: store straight into it as f32.
            p.out_bf16 = 0; p.epi = EpiChain{}; p.n_dst = 1; p.ldc = static_cast<long long>(ld_partial);
        }
        // Epilogue through TMA stores when there is one plain destination the TMA unit can address; peers and
        // split-K slabs keep the warp-issued stores.
        CUtensorMap tc = ta;
        {
            const uint32_t oelem = p.out_bf16 ? 2u : 4u;
            // TMA clips a store at the tensor edge in 16-byte units, so N must be a whole number of them for
            // nothing beyond column N to be touched.
            p.cluster_sk = cluster_sk ? static_cast<int>(sk) : 0;
            const bool ok = !to_slabs && p.n_dst == 1 && (g.c_dst[0] % 16 == 0) && ((static_cast<uint64_t>(p.ldc) * oelem) % 16 == 0) &&
                            ((static_cast<uint64_t>(g.n) * oelem) % 16 == 0);
            p.tma_store = 0;
            if (ok) {
                rc = get_tmap(ctx, g.c_dst[0], g.n, g.m, static_cast<uint64_t>(p.ldc), p.out_bf16 ? 32 : 16, 32, &tc, oelem);   // 64-byte rows
                if (rc != T0B_OK) return rc;
                p.tma_store = 1;
            }
        }
        const int num_work = p.tiles_m * p.tiles_n * p.split_k;
#ifdef T0B_TRACE
        p.trace = nullptr;
        if (ctx->trace_buf && ctx->trace_slots > 0 && (cluster_sk ? num_work : ctx->num_sms) <= kTraceCtas) {
            p.trace = reinterpret_cast<unsigned long long*>(ctx->trace_buf) +
                      static_cast<size_t>(ctx->trace_next % ctx->trace_slots) * kTraceCtas * 16;
            ++ctx->trace_next;
        }
#endif
        if (g.accumulate || g.dyn_rows || g.late_wait) {
            KernelParams<2> q{};
            static_cast<GemmParams&>(q) = p;
            q.inner.dyn_rows = g.dyn_rows; q.inner.dyn_off = g.dyn_off; q.inner.dyn_k = g.dyn_k;
            q.inner.accumulate = g.accumulate ? 1 : 0;
            q.inner.late_wait = g.late_wait ? 1 : 0;
            rc = launch_plan<2>(ctx, plan, ta, tb, tc, q, num_work);
        } else {
            rc = launch_plan<0>(ctx, plan, ta, tb, tc, p, num_work);
        }
        if (rc != T0B_OK) return rc;
        ++ctx->launches;
    }

    if (!g.slabs_only && sk > 1 && !cluster_sk) {
        for (int d = 0; d < g.n_dst; ++d) {
            int32_t rc = launch_reduce(ctx, partial, sk, g.m, g.n, slab_stride, ld_partial, ld_partial == pitch4, reinterpret_cast<void*>(g.c_dst[d]),
                                       g.ldc, g.out_bf16, g.epi);
            if (rc != T0B_OK) return rc;
            ++ctx->launches;
        }
    }
    return T0B_OK;
}

// Pseudo-random bf16 fill for the tuner: operands of zeros would draw less power than real data and make the
// measured clocks (and the ranking of configs) unrepresentative.
__global__ void __launch_bounds__(256) fill_random_bf16_kernel(__nv_bfloat16* dst, size_t n, uint32_t seed, float scale) {
    const size_t stride = static_cast<size_t>(gridDim.x) * blockDim.x;
    for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < n; i += stride) {
        uint32_t x = static_cast<uint32_t>(i) * 2654435761u ^ seed;
        x ^= x >> 16; x *= 0x7feb352du; x ^= x >> 15; x *= 0x846ca68bu; x ^= x >> 16;
        const float u = static_cast<float>(x >> 8) * (1.0f / 8388608.0f) - 1.0f;   // [-1, 1)
        dst[i] = __float2bfloat16_rn(u * scale);
    }
}

GemmCall call_of(const InnerGemm& d) {
    GemmCall g{};
    g.trans_a = d.trans_a; g.trans_b = d.trans_b; g.a = d.a; g.b = d.b;
    g.c_dst[0] = d.c; g.n_dst = 1; g.m = d.m; g.n = d.n; g.k = d.k; g.lda = d.lda; g.ldb = d.ldb; g.ldc = d.ldc;
    g.out_bf16 = d.out_bf16; g.accumulate = d.accumulate; g.workspace = d.slabs; g.workspace_bytes = d.slab_bytes;
    g.dyn_rows = reinterpret_cast<const int*>(d.dyn_rows); g.dyn_off = d.dyn_off; g.dyn_k = d.dyn_k;
    g.late_wait = d.late_wait;
    return g;
}

uint32_t rd_u32(const uint8_t* p) { return p[0] | (p[1] << 8) | (p[2] << 16) | (static_cast<uint32_t>(p[3]) << 24); }
uint64_t rd_u64(const uint8_t* p) { return rd_u32(p) | (static_cast<uint64_t>(rd_u32(p + 4)) << 32); }

}  // namespace

namespace {
// Tiles and splits of the two gradient products of a head, where the caller has not measured any (t0b_tune, the shipped table).
// The head's own gradient is a huge output of a contraction over the rows of a batch, never split; the hidden states' gradient
// is a small output of a contraction over the vocabulary, split until the SMs have work.  The cost model of t0b_gemm is made for
// neither: here a wave costs what its stores or its operands from L2 cost, whichever is more, and K may be cut into up to 32
// ranges.  Cycles measured at (m, n, k) = 32000 x 1024 x 128, 50257 x 1000 x 777, 4096 x 32000 x 1024: with k = 128, 128x256
// tiles take 19.6 us against 25.2 for 256x512; with k = 777, 122 us against 101 for 256x256 and 96 for 256x512.
t0b_gemm_config head_grad_config(t0b_ctx* ctx, const GemmCall& g, bool split) {
    struct Cand { const char* name; uint32_t bm, bn, cg; double kb_cycles, epi, floor; };
    static const Cand cands[] = {{"b200_256x512", 256, 512, 2, 1165.0, 10500.0, 0.0}, {"b200_256x256", 256, 256, 2, 830.0, 0.0, 6500.0},
                                 {"b200_128x256", 128, 256, 1, 1000.0, 0.0, 4900.0},  {"b200_128x128", 128, 128, 1, 700.0, 0.0, 3000.0},
                                 {"b200_128x64", 128, 64, 1, 550.0, 0.0, 2500.0}};
    const uint32_t kb = (g.k + 63) / 64;
    const Cand* best = nullptr;
    uint32_t best_sk = 1;
    double best_cost = 1e300;
    for (const Cand& c : cands) {
        const uint64_t tiles = static_cast<uint64_t>((g.m + c.bm - 1) / c.bm) * ((g.n + c.bn - 1) / c.bn), clusters = static_cast<uint64_t>(ctx->num_sms) / c.cg;
        for (uint32_t sk = 1; sk <= (split ? 32u : 1u); sk *= 2) {
            if (sk > 1 && (kb / sk < 4 || tiles * (sk / 2) >= clusters)) break;   // split only while SMs are idle
            double cost = static_cast<double>((tiles * sk + clusters - 1) / clusters) * std::max((kb + sk - 1) / sk * c.kb_cycles + c.epi, c.floor);
            // The sum over the ranges: inside a cluster over distributed shared memory, or through slabs and a second kernel.
            if (sk > 1) cost += (c.cg == 1 && (sk <= 4 || (sk == 8 && tiles <= 15))) ? 7000.0 : 8000.0 + 100.0 * sk + static_cast<double>(g.m) * g.n * 4.0 * (sk + 1) / 3300.0;
            if (cost < best_cost) {
                best_cost = cost;
                best = &c;
                best_sk = sk;
            }
        }
    }
    t0b_gemm_config cfg{};
    t0b_config_preset(best->name, &cfg);
    cfg.swap_grid = g.m >= g.n ? 1 : 0;
    cfg.split_k = best_sk > 1 ? best_sk : 0;
    return cfg;
}

// The config of an inner product: what was measured for it, else the rule above.
int32_t inner_config(t0b_ctx* ctx, const InnerGemm& d, const GemmCall& g, t0b_gemm_config* cfg) {
    int source = 0;
    const char* from = "";
    if (!ctx->force_config.empty()) {
        const int32_t rc = choose_config(ctx, g, cfg, &from);
        if (rc != T0B_OK) return rc;
    } else if (!tuned_lookup(g.m, g.n, g.k, g.trans_a, g.trans_b, g.out_bf16, cfg, &source)) {
        *cfg = head_grad_config(ctx, g, !d.head_grad);
    }
    if (d.head_grad || g.accumulate) cfg->split_k = 0;
    return T0B_OK;
}

}  // namespace

namespace t0b {

size_t inner_gemm_slab_bytes(t0b_ctx* ctx, const InnerGemm& d) {
    const GemmCall g = call_of(d);
    t0b_gemm_config cfg;
    if (inner_config(ctx, d, g, &cfg) != T0B_OK || cfg.split_k <= 1) return 0;
    t0b_gemm_plan plan;
    const PlanInput pin{g.m, g.n, g.k, g.trans_a, g.trans_b, g.lda, g.ldb, g.a, g.b, ctx->num_sms};
    resolve_plan(&cfg, pin, &plan);
    if (plan.split_k <= 1 || splitk_in_cluster(ctx, g, plan)) return 0;
    return static_cast<size_t>(plan.split_k) * g.m * slab_pitch(g.n) * 4;
}

int32_t inner_gemm(t0b_ctx* ctx, const InnerGemm& d) {
    GemmCall g = call_of(d);
    t0b_gemm_config cfg;
    const int32_t rc = inner_config(ctx, d, g, &cfg);
    if (rc != T0B_OK) return rc;
    // The caller's slabs were sized for the config of that moment; a table entry that appeared since may want more.  The
    // context's own workspace is never used here: it may be freed by a later call while a captured graph still holds it.
    if (cfg.split_k > 1 && inner_gemm_slab_bytes(ctx, d) > d.slab_bytes) cfg.split_k = 0;
    g.cfg = &cfg;
    return run_gemm(ctx, g);
}

HeadPlan head_plan(t0b_ctx* ctx, uint32_t rows, uint32_t vocab, uint32_t dim) {
    // The three tiles of the softmax epilogue by waves and cycles per 64-deep K block, or per epilogue where that is more: a CTA
    // pair shares each block of head columns between 256 rows; a single CTA takes 128 rows, in 256 or 128 columns, and needs
    // 1.5 times the operand bytes from L2 for the same products (777 x 1000 -> 50257: 129 us against the pair's 101 us, although
    // the pair's last rows are padding; 16 x 1024 -> 32000: 18.7 us against 22.1 us).
    struct Cand { uint32_t bm, bn, cg; double kb_cycles, epi_cycles; };
    static const Cand cands[] = {{256, 256, 2, 800.0, 5000.0}, {128, 256, 1, 900.0, 5000.0}, {128, 128, 1, 700.0, 2800.0}};
    const double kb = (dim + 63) / 64;
    HeadPlan best{};
    double best_cost = 1e300;
    for (const Cand& c : cands) {
        const uint64_t tiles = static_cast<uint64_t>((rows + c.bm - 1) / c.bm) * ((vocab + c.bn - 1) / c.bn);
        const uint64_t clusters = static_cast<uint64_t>(ctx->num_sms) / c.cg;
        const double waves = static_cast<double>((tiles + clusters - 1) / clusters);
        const double cost = waves * std::max(kb * c.kb_cycles, c.epi_cycles) + c.epi_cycles;
        if (cost < best_cost) {
            best_cost = cost;
            best.bm = c.bm; best.bn = c.bn; best.cta_group = c.cg;
            best.part_cols = c.bn / 2;
        }
    }
    return best;
}

int32_t head_gemm(t0b_ctx* ctx, const HeadGemm& d) {
    const HeadPlan& plan = d.plan;
    CUtensorMap ta, tb, tc;
    int32_t rc = get_tmap(ctx, d.x, d.dim, d.rows, d.ldx, 64, 128, &ta);
    if (rc != T0B_OK) return rc;
    if (d.trans_w) rc = get_tmap(ctx, d.w, d.dim, d.vocab, d.ldw, 64, plan.bn / plan.cta_group, &tb);
    else rc = get_tmap(ctx, d.w, d.vocab, d.dim, d.ldw, 64, 64, &tb);
    if (rc != T0B_OK) return rc;
    tc = ta;
    if (d.u) {
        rc = get_tmap(ctx, d.u, d.ldu, d.rows, d.ldu, 32, 32, &tc);   // 16-bit elements, moved as they are
        if (rc != T0B_OK) return rc;
    }
    KernelParams<1> p{};
    p.n_dst = 1;
    p.M = static_cast<int>(d.rows); p.N = static_cast<int>(d.vocab); p.K = static_cast<int>(d.dim);
    p.tiles_m = static_cast<int>((d.rows + plan.bm - 1) / plan.bm);
    p.tiles_n = static_cast<int>((d.vocab + plan.bn - 1) / plan.bn);
    p.split_k = 1;
    p.kb_total = static_cast<int>((d.dim + 63) / 64);
    p.kb_per_split = p.kb_total;
    p.b_mn_major = d.trans_w ? 0 : 1;
    p.raster_along_n = d.rows >= d.vocab ? 0 : 1;
    p.group = raster_group(ctx, plan.bm, plan.bn, plan.cta_group, d.rows >= d.vocab);
    p.mn_lbo = 8192; p.mn_sbo = 1024; p.mn_kstep = 2048;
    p.status = ctx->status_dev;
    p.wait_limit_ns = ctx->wait_limit_ns;
    p.wait_hint_ns = ctx->wait_hint_ns;
    p.tma_store = d.u ? 1 : 0;
    p.head.part = reinterpret_cast<float2*>(d.part);
    p.head.part_ld = static_cast<long long>(d.part_ld);
    p.head.c = d.c;
    p.head.ids = reinterpret_cast<const uint32_t*>(d.ids);
    p.head.row_of = reinterpret_cast<const uint32_t*>(d.row_of);
    p.inner.dyn_rows = reinterpret_cast<const int*>(d.dyn_rows);
    p.inner.dyn_off = d.dyn_off;
    p.head.n_ids = static_cast<int>(d.n_ids);
    p.head.z_sel = reinterpret_cast<float*>(d.z_sel);
    p.head.store_u = d.u ? 1 : 0;
    const int num_work = p.tiles_m * p.tiles_n;
    if (plan.cta_group == 2) rc = launch_variant<256, 2, 1, 0, 1>(ctx, ta, tb, tc, p, num_work);
    else if (plan.bn == 256) rc = launch_variant<256, 1, 1, 0, 1>(ctx, ta, tb, tc, p, num_work);
    else rc = launch_variant<128, 1, 1, 0, 1>(ctx, ta, tb, tc, p, num_work);
    if (rc == T0B_OK) ++ctx->launches;
    return rc;
}

}  // namespace t0b

extern "C" {

int32_t t0b_trace_set(t0b_ctx* ctx, uint64_t buf, uint32_t launches) {
    int32_t rc = precheck(ctx);
    if (rc != T0B_OK) return rc;
#ifdef T0B_TRACE
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    ctx->trace_buf = buf;
    ctx->trace_slots = buf ? launches : 0;
    ctx->trace_next = 0;
    return T0B_OK;
#else
    (void)buf; (void)launches;
    return set_error(ctx, T0B_ERR_UNSUPPORTED, "trace_set: this is the regular build; the timeline build is libt0b200_trace.so");
#endif
}

int32_t t0b_gemm(t0b_ctx* ctx, const t0b_gemm_config* cfg, int32_t trans_a, int32_t trans_b, uint64_t a, uint64_t b,
                 uint64_t c, uint32_t m, uint32_t n, uint32_t k, uint64_t lda, uint64_t ldb, uint64_t ldc,
                 int32_t out_dtype, int32_t epilogue, uint64_t bias, float alpha, uint64_t workspace,
                 size_t workspace_bytes, int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    GemmCall g{};
    g.cfg = cfg; g.trans_a = trans_a != 0; g.trans_b = trans_b != 0; g.a = a; g.b = b;
    g.c_dst[0] = c; g.n_dst = 1; g.m = m; g.n = n; g.k = k; g.lda = lda; g.ldb = ldb; g.ldc = ldc;
    g.out_bf16 = out_dtype == T0B_OUT_BF16;
    g.workspace = workspace; g.workspace_bytes = workspace_bytes;
    if (out_dtype != T0B_OUT_F32 && out_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "gemm: unknown out_dtype %d", out_dtype);
    rc = make_chain(ctx, &epilogue, 1, bias, alpha, 0.0f, 0.0f, &g.epi);
    if (rc != T0B_OK) return rc;
    rc = run_gemm(ctx, g);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_gemm", 0);
}

int32_t t0b_gemm_chain(t0b_ctx* ctx, const t0b_gemm_config* cfg, int32_t trans_a, int32_t trans_b, uint64_t a, uint64_t b,
                       uint64_t c, uint32_t m, uint32_t n, uint32_t k, uint64_t lda, uint64_t ldb, uint64_t ldc,
                       int32_t out_dtype, const int32_t* ops, int32_t n_ops, uint64_t bias, float scale, float clamp_min,
                       float clamp_max, uint64_t workspace, size_t workspace_bytes, int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (n_ops < 0 || (n_ops > 0 && !ops)) return set_error(ctx, T0B_ERR_INVALID, "gemm_chain: bad operation list");
    if (out_dtype != T0B_OUT_F32 && out_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "gemm: unknown out_dtype %d", out_dtype);
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    GemmCall g{};
    g.cfg = cfg; g.trans_a = trans_a != 0; g.trans_b = trans_b != 0; g.a = a; g.b = b;
    g.c_dst[0] = c; g.n_dst = 1; g.m = m; g.n = n; g.k = k; g.lda = lda; g.ldb = ldb; g.ldc = ldc;
    g.out_bf16 = out_dtype == T0B_OUT_BF16;
    g.workspace = workspace; g.workspace_bytes = workspace_bytes;
    rc = make_chain(ctx, ops, n_ops, bias, scale, clamp_min, clamp_max, &g.epi);
    if (rc != T0B_OK) return rc;
    rc = run_gemm(ctx, g);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_gemm_chain", 0);
}

int32_t t0b_gemm_host(t0b_ctx* ctx, const t0b_gemm_config* cfg, int32_t trans_a, int32_t trans_b, const void* a, const void* b,
                      void* c, uint32_t m, uint32_t n, uint32_t k, uint64_t lda, uint64_t ldb, uint64_t ldc, int32_t out_dtype,
                      uint32_t chunk_rows) {
    int32_t rc = precheck(ctx);
    if (rc != T0B_OK) return rc;
    if (m == 0 || n == 0) return T0B_OK;
    if (!a || !b || !c) return set_error(ctx, T0B_ERR_INVALID, "gemm_host: null host pointer");
    if (out_dtype != T0B_OUT_F32 && out_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "gemm_host: unknown out_dtype %d", out_dtype);
    const uint64_t a_rows = trans_a ? k : m, a_cols = trans_a ? m : k;
    const uint64_t b_rows = trans_b ? n : k, b_cols = trans_b ? k : n;
    if (lda < a_cols || ldb < b_cols || ldc < n) return set_error(ctx, T0B_ERR_INVALID, "gemm_host: pitch smaller than the row");
    if (ctx->capturing) return set_error(ctx, T0B_ERR_INVALID, "gemm_host: not available during graph capture");
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    if (!ctx->h2d_stream) {
        rc = check_cuda(ctx, cudaStreamCreateWithFlags(&ctx->h2d_stream, cudaStreamNonBlocking), "cudaStreamCreate(h2d)");
        if (rc == T0B_OK) rc = check_cuda(ctx, cudaStreamCreateWithFlags(&ctx->d2h_stream, cudaStreamNonBlocking), "cudaStreamCreate(d2h)");
        if (rc != T0B_OK) return rc;
    }
    const size_t oelem = out_dtype == T0B_OUT_BF16 ? 2 : 4;
    // Device copies are dense, with pitches rounded up so that every row starts on a 16-byte boundary (TMA).
    const uint64_t dlda = (a_cols + 7) & ~7ull, dldb = (b_cols + 7) & ~7ull, dldc = (static_cast<uint64_t>(n) + 7) & ~7ull;
    uint64_t da = 0, db = 0, dc = 0;
    rc = t0b_alloc(ctx, a_rows * dlda * 2, &da);
    if (rc == T0B_OK) rc = t0b_alloc(ctx, b_rows * dldb * 2, &db);
    if (rc == T0B_OK) rc = t0b_alloc(ctx, static_cast<uint64_t>(m) * dldc * oelem, &dc);
    if (rc != T0B_OK) {
        if (da) t0b_recycle(ctx, da);
        if (db) t0b_recycle(ctx, db);
        return rc;
    }
    // The product is cut into row blocks of A (and C) and column panels of B (and C).  Step s uploads A block s and
    // B panel s; the blocks of C that became computable (row strip s up to panel s, column strip s above it) are
    // multiplied and copied back while step s+1 uploads, so both PCIe directions stay busy from the second step on.
    if (chunk_rows == 0) chunk_rows = std::max<uint32_t>(512u, ((m + 7) / 8 + 511u) & ~511u);   // about eight blocks
    chunk_rows = (chunk_rows + 127u) & ~127u;
    const uint32_t nchunks = (m + chunk_rows - 1) / chunk_rows;
    uint32_t want_panels = std::max(1u, std::min(8u, n / 512u));
    if (const char* e = std::getenv("T0B_HOST_PANELS")) want_panels = std::max(1, std::atoi(e));   // measurement knob
    const uint32_t panel_cols = (((n + want_panels - 1) / want_panels) + 63u) & ~63u;
    const uint32_t npanels = (n + panel_cols - 1) / panel_cols;
    const uint32_t nsteps = std::max(nchunks, npanels);
    std::vector<cudaEvent_t> ev(3 * static_cast<size_t>(nsteps) + 1, nullptr);
    for (auto& x : ev) cudaEventCreateWithFlags(&x, cudaEventDisableTiming);
    cudaEvent_t* ev_up = ev.data();                  // step s uploaded
    cudaEvent_t* ev_row = ev.data() + nsteps;        // row strip s multiplied
    cudaEvent_t* ev_col = ev.data() + 2 * nsteps;    // column strip s multiplied
    cudaEvent_t ev_start = ev.back();
    // Work already queued on the compute stream (e.g. earlier users of the pooled buffers) goes first.
    cudaEventRecord(ev_start, ctx->stream);
    cudaStreamWaitEvent(ctx->h2d_stream, ev_start, 0);
    cudaStreamWaitEvent(ctx->d2h_stream, ev_start, 0);
    cudaError_t e = cudaSuccess;
    GemmCall g{};
    g.cfg = cfg; g.trans_a = trans_a != 0; g.trans_b = trans_b != 0; g.n_dst = 1;
    g.k = k; g.lda = dlda; g.ldb = dldb; g.ldc = dldc; g.out_bf16 = out_dtype == T0B_OUT_BF16;
    g.no_auto_split = true;   // blocks of one product must not differ in summation order; the call is PCIe-bound anyway
    // Multiply C[r0:r0+rows, c0:c0+cols] on the compute stream, then copy it back behind `done`.
    auto strip = [&](uint32_t r0, uint32_t rows, uint32_t c0, uint32_t cols, cudaEvent_t done) {
        g.a = trans_a ? da + static_cast<uint64_t>(r0) * 2 : da + static_cast<uint64_t>(r0) * dlda * 2;
        g.b = trans_b ? db + static_cast<uint64_t>(c0) * dldb * 2 : db + static_cast<uint64_t>(c0) * 2;
        g.c_dst[0] = dc + (static_cast<uint64_t>(r0) * dldc + c0) * oelem;
        g.m = rows;
        g.n = cols;
        rc = run_gemm(ctx, g);
        if (rc != T0B_OK) return;
        cudaEventRecord(done, ctx->stream);
        cudaStreamWaitEvent(ctx->d2h_stream, done, 0);
        e = cudaMemcpy2DAsync(static_cast<char*>(c) + (static_cast<uint64_t>(r0) * ldc + c0) * oelem, ldc * oelem,
                              reinterpret_cast<char*>(dc) + (static_cast<uint64_t>(r0) * dldc + c0) * oelem, dldc * oelem,
                              static_cast<size_t>(cols) * oelem, rows, cudaMemcpyDeviceToHost, ctx->d2h_stream);
    };
    for (uint32_t s = 0; s < nsteps && e == cudaSuccess && rc == T0B_OK; ++s) {
        const uint32_t r0 = s * chunk_rows, c0 = s * panel_cols;
        const uint32_t rows = s < nchunks ? std::min(chunk_rows, m - r0) : 0;
        const uint32_t cols = s < npanels ? std::min(panel_cols, n - c0) : 0;
        if (rows && e == cudaSuccess) {
            if (!trans_a)   // A[M, K]: a row block
                e = cudaMemcpy2DAsync(reinterpret_cast<char*>(da) + static_cast<uint64_t>(r0) * dlda * 2, dlda * 2,
                                      static_cast<const char*>(a) + static_cast<uint64_t>(r0) * lda * 2, lda * 2,
                                      static_cast<size_t>(k) * 2, rows, cudaMemcpyHostToDevice, ctx->h2d_stream);
            else            // A[K, M]: a column block
                e = cudaMemcpy2DAsync(reinterpret_cast<char*>(da) + static_cast<uint64_t>(r0) * 2, dlda * 2,
                                      static_cast<const char*>(a) + static_cast<uint64_t>(r0) * 2, lda * 2,
                                      static_cast<size_t>(rows) * 2, k, cudaMemcpyHostToDevice, ctx->h2d_stream);
        }
        if (cols && e == cudaSuccess) {
            if (!trans_b)   // B[K, N]: a column block
                e = cudaMemcpy2DAsync(reinterpret_cast<char*>(db) + static_cast<uint64_t>(c0) * 2, dldb * 2,
                                      static_cast<const char*>(b) + static_cast<uint64_t>(c0) * 2, ldb * 2,
                                      static_cast<size_t>(cols) * 2, k, cudaMemcpyHostToDevice, ctx->h2d_stream);
            else            // B[N, K]: a row block
                e = cudaMemcpy2DAsync(reinterpret_cast<char*>(db) + static_cast<uint64_t>(c0) * dldb * 2, dldb * 2,
                                      static_cast<const char*>(b) + static_cast<uint64_t>(c0) * ldb * 2, ldb * 2,
                                      static_cast<size_t>(k) * 2, cols, cudaMemcpyHostToDevice, ctx->h2d_stream);
        }
        if (e != cudaSuccess) break;
        cudaEventRecord(ev_up[s], ctx->h2d_stream);
        cudaStreamWaitEvent(ctx->stream, ev_up[s], 0);
        // Row strip: the new rows against every panel uploaded so far.
        if (rows) {
            const uint32_t last_panel = std::min(s, npanels - 1);
            const uint32_t c_end = std::min(n, (last_panel + 1) * panel_cols);
            strip(r0, rows, 0, c_end, ev_row[s]);
        }
        // Column strip: the new panel against every row block uploaded before this step.
        if (cols && s > 0 && e == cudaSuccess && rc == T0B_OK) {
            const uint32_t last_chunk = std::min(s - 1, nchunks - 1);
            const uint32_t r_end = std::min(m, (last_chunk + 1) * chunk_rows);
            strip(0, r_end, c0, cols, ev_col[s]);
        }
    }
    cudaError_t e1 = cudaStreamSynchronize(ctx->d2h_stream);
    cudaError_t e2 = cudaStreamSynchronize(ctx->stream);
    cudaError_t e3 = cudaStreamSynchronize(ctx->h2d_stream);
    for (auto& x : ev) cudaEventDestroy(x);
    t0b_recycle(ctx, da);
    t0b_recycle(ctx, db);
    t0b_recycle(ctx, dc);
    if (rc != T0B_OK) return rc;
    for (cudaError_t x : {e, e1, e2, e3})
        if (x != cudaSuccess) return check_cuda(ctx, x, "gemm_host");
    const int st = take_device_status(ctx);
    if (st != 0) return set_error(ctx, T0B_ERR_DEVICE, "gemm_host: device status %d (a bounded in-kernel wait ran out)", st);
    return T0B_OK;
}

int32_t t0b_multi_dst_config(uint32_t m, uint32_t k, uint32_t n_local, int32_t n_dst, int32_t num_sms, t0b_gemm_config* out) {
    if (!out || n_dst < 1 || n_dst > kMaxDst) return T0B_ERR_INVALID;
    // The measured config of this rank's block (row-major operands, bf16 output: the sharded benchmark's layout), else
    // the cost model.
    if (!tuned_lookup(m, n_local, k, 0, 0, 1, out, nullptr)) default_b200_config(m, k, n_local, num_sms > 0 ? num_sms : 148, out);
    // Stores to a peer retire at the NVLink rate (about 0.7 TB/s for SM-issued stores, measured), far below the rate the
    // epilogue can issue them, so the epilogue warps of a tile block in stores for as long as the tile's share of the link
    // time.  The tiles that keep both TMEM accumulators for one tile (256x512, 512x256) are the fastest at the math but
    // cannot start the next main loop until that epilogue is over; the 256x256 tile double-buffers its accumulators, so
    // the stores of tile i retire while tile i+1 is multiplied.  It pays once the link time is a sizeable part of the
    // math time: measured on the 32768 x (32768/G) x 8192 blocks, two GPUs (link / math = 0.25) run 12 % faster on
    // 256x512, four and eight GPUs (0.75 and 1.8) on 256x256.
    if (n_dst > 1 && (out->tile_m >= 512 || out->tile_n >= 512)) {
        const double link_s = static_cast<double>(n_dst - 1) * m * n_local * 2.0 / 0.70e12;   // bf16 output assumed
        const double math_s = 2.0 * m * static_cast<double>(n_local) * k / 1.45e15;
        if (link_s > 0.5 * math_s) {
            out->tile_m = 256;
            out->tile_n = 256;
            out->wg_size = 192;
        }
    }
    out->split_k = 0;   // the fused store writes final values; there is no slab stage
    return T0B_OK;
}

int32_t t0b_gemm_multi_dst(t0b_ctx* ctx, const t0b_gemm_config* cfg, int32_t trans_a, int32_t trans_b, uint64_t a,
                           uint64_t b, const uint64_t* c_dsts, int32_t n_dst, uint32_t m, uint32_t n_local, uint32_t k,
                           uint64_t lda, uint64_t ldb, uint64_t ldc, uint64_t col0, int32_t out_dtype, int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (!c_dsts || n_dst < 1 || n_dst > kMaxDst) return set_error(ctx, T0B_ERR_INVALID, "gemm_multi_dst: 1..%d destinations", kMaxDst);
    if (col0 + n_local > ldc) return set_error(ctx, T0B_ERR_INVALID, "gemm_multi_dst: column block exceeds the row pitch");
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    GemmCall g{};
    t0b_gemm_config local;
    if (cfg) {
        local = *cfg;
        local.split_k = 0;   // the fused store writes final values; no slab stage
        g.cfg = &local;
    } else {
        t0b_multi_dst_config(m, k, n_local, n_dst, ctx->num_sms, &local);
        g.cfg = &local;
    }
    g.trans_a = trans_a != 0; g.trans_b = trans_b != 0; g.a = a; g.b = b;
    const size_t elem = out_dtype == T0B_OUT_BF16 ? 2 : 4;
    for (int d = 0; d < n_dst; ++d) g.c_dst[d] = c_dsts[d] ? c_dsts[d] + col0 * elem : 0;
    g.n_dst = n_dst; g.m = m; g.n = n_local; g.k = k; g.lda = lda; g.ldb = ldb; g.ldc = ldc;
    g.out_bf16 = out_dtype == T0B_OUT_BF16;
    rc = run_gemm(ctx, g);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_gemm_multi_dst", 0);
}

int32_t t0b_gemm_slabs(t0b_ctx* ctx, const t0b_gemm_config* cfg, uint64_t x, uint64_t wt, uint64_t y, uint32_t m,
                       uint32_t n, uint32_t k, uint32_t split_k, int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (split_k == 0 || (split_k & (split_k - 1)) != 0)
        return set_error(ctx, T0B_ERR_INVALID, "gemm_slabs: split_k=%u must be a power of 2", split_k);
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    t0b_gemm_config local;
    if (cfg) local = *cfg;
    else default_b200_config(m, k, n, ctx->num_sms, &local);
    GemmCall g{};
    g.cfg = &local; g.trans_a = 0; g.trans_b = 1; g.a = x; g.b = wt; g.c_dst[0] = y; g.n_dst = 1;
    g.m = m; g.n = n; g.k = k; g.lda = k; g.ldb = k; g.ldc = n; g.out_bf16 = 0;
    g.slabs_only = true; g.force_split = split_k;
    rc = run_gemm(ctx, g);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_gemm_slabs", 0);
}

int32_t t0b_splitk_reduce(t0b_ctx* ctx, uint64_t partial, uint32_t split_k, uint32_t m, uint32_t n,
                          uint64_t slab_stride_elems, uint64_t ld_partial, uint64_t c, uint64_t ldc, int32_t out_dtype,
                          int32_t epilogue, uint64_t bias, float alpha, int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (!partial || !c || split_k == 0) return set_error(ctx, T0B_ERR_INVALID, "splitk_reduce: null pointer or zero split");
    if (m == 0 || n == 0) return T0B_OK;
    if (ld_partial < n || ldc < n) return set_error(ctx, T0B_ERR_INVALID, "splitk_reduce: pitch smaller than n");
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    EpiChain chain;
    rc = make_chain(ctx, &epilogue, 1, bias, alpha, 0.0f, 0.0f, &chain);
    if (rc != T0B_OK) return rc;
    rc = launch_reduce(ctx, reinterpret_cast<const float*>(partial), split_k, m, n, slab_stride_elems, ld_partial, false,
                       reinterpret_cast<void*>(c), ldc, out_dtype == T0B_OUT_BF16, chain);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_splitk_reduce", 1);
}

int32_t t0b_dispatch_kernargs(t0b_ctx* ctx, const t0b_gemm_config* cfg, uint32_t grid_x, uint32_t grid_y,
                              const uint8_t* ka, size_t len, int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (!cfg || !ka) return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: null config or kernargs");
    if (len != 40 && len != 44 && len != 48)
        return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: kernarg blob must be 40, 44 or 48 bytes, got %zu", len);
    if (cfg->wg_size == 0 || cfg->tile_m == 0 || cfg->tile_n == 0)
        return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: config with zero tile or workgroup size");
    const uint64_t x = rd_u64(ka), wt = rd_u64(ka + 8), y = rd_u64(ka + 16);
    const uint32_t k = rd_u32(ka + 24), n_pitch = rd_u32(ka + 28), y_stride = rd_u32(ka + 36);
    const uint32_t sk = cfg->split_k > 1 ? cfg->split_k : 1;
    if (grid_x % cfg->wg_size != 0) return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: grid_x is not a multiple of wg_size");
    const uint32_t fast_tiles = grid_x / cfg->wg_size;
    if (grid_y % sk != 0) return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: grid_y is not a multiple of split_k");
    const uint32_t slow_tiles = grid_y / sk;
    const uint32_t tiles_m = cfg->swap_grid ? slow_tiles : fast_tiles;
    const uint32_t tiles_n = cfg->swap_grid ? fast_tiles : slow_tiles;
    const uint32_t eff_n = cfg->tile_n * std::max(1u, cfg->n_col_passes);
    uint32_t m, n;
    if (len == 44) {
        m = rd_u32(ka + 40);                                 // the tile_ir blob carries M
        n = std::min(n_pitch, tiles_n * eff_n);
        if (m > tiles_m * cfg->tile_m) return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: M exceeds the grid");
    } else {
        m = tiles_m * cfg->tile_m;                           // recovered from the grid
        n = tiles_n * eff_n;
        if (n > n_pitch) return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: grid covers more columns than the N kernarg");
    }
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    GemmCall g{};
    t0b_gemm_config local = *cfg;
    g.cfg = &local; g.trans_a = 0; g.trans_b = 1; g.a = x; g.b = wt; g.c_dst[0] = y; g.n_dst = 1;
    g.m = m; g.n = n; g.k = k; g.lda = k; g.ldb = k; g.ldc = n_pitch;
    g.out_bf16 = 0;
    {
        int32_t epi = static_cast<int32_t>(cfg->epilogue);
        const uint64_t bias = len == 48 ? rd_u64(ka + 40) : 0;
        if (epi != EPI_STORE && (len != 48 || !bias)) epi = EPI_STORE;   // gemm_gen.rs:437: bias 0 = plain store
        if (sk > 1) epi = EPI_STORE;
        rc = make_chain(ctx, &epi, 1, bias, 1.0f, 0.0f, 0.0f, &g.epi);
        if (rc != T0B_OK) return rc;
    }
    if (sk > 1) {
        if (y_stride != m * n * 4u)
            return set_error(ctx, T0B_ERR_INVALID, "dispatch_kernargs: y_split_stride %u does not match M*N*4 = %u", y_stride, m * n * 4u);
        g.slabs_only = true; g.force_split = sk; g.ldc = n;
    } else {
        local.split_k = 0;
    }
    rc = run_gemm(ctx, g);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_dispatch_kernargs", 0);
}

int32_t t0b_tile_dispatch(t0b_ctx* ctx, const t0b_tile_gemm* spec, const uint32_t grid[3], const uint8_t* ka, size_t len,
                          int32_t async) {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (!spec || !grid || !ka) return set_error(ctx, T0B_ERR_INVALID, "tile_dispatch: null spec, grid or kernargs");
    if (!tile_spec_valid(spec)) return set_error(ctx, T0B_ERR_INVALID, "tile_dispatch: invalid TileGemm spec");
    size_t bias_off = 0, scale_off = 0, clamp_off = 0;
    const size_t want = tile_kernarg_layout(spec, &bias_off, &scale_off, &clamp_off);
    if (len != want)
        return set_error(ctx, T0B_ERR_INVALID, "tile_dispatch: this spec takes a %zu-byte kernarg blob, got %zu", want, len);
    const uint64_t x = rd_u64(ka), wt = rd_u64(ka + 8), y = rd_u64(ka + 16);
    const uint32_t k = rd_u32(ka + 24), n = rd_u32(ka + 28), m = rd_u32(ka + 40);
    uint32_t expect[3];
    t0b_tile_compute_grid(spec, m, n, expect);
    if (grid[0] != expect[0] || grid[1] != expect[1] || grid[2] != 1)
        return set_error(ctx, T0B_ERR_INVALID, "tile_dispatch: grid [%u,%u,%u] does not match compute_grid [%u,%u,1] for M=%u N=%u",
                         grid[0], grid[1], grid[2], expect[0], expect[1], m, n);
    uint64_t bias = 0;
    float scale = 1.0f, clamp_min = 0.0f, clamp_max = 0.0f;
    if (bias_off) {
        bias = rd_u64(ka + bias_off);
        if (!bias) return set_error(ctx, T0B_ERR_INVALID, "tile_dispatch: the epilogue has BiasAdd but the bias pointer is null");
    }
    auto rd_f32 = [&](size_t off) { uint32_t u = rd_u32(ka + off); float f; std::memcpy(&f, &u, 4); return f; };
    if (scale_off) scale = rd_f32(scale_off);
    if (clamp_off) { clamp_min = rd_f32(clamp_off); clamp_max = rd_f32(clamp_off + 4); }

    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    // The spec's tile becomes a B200 tile the same way a GemmConfig's does (resolve_plan).
    t0b_gemm_config cfg{};
    cfg.tile_m = spec->tile_m; cfg.tile_n = spec->tile_n; cfg.tile_k = spec->tile_k;
    cfg.wg_size = t0b_tile_wg_size(spec); cfg.use_lds = 1; cfg.double_buffer = spec->double_buffer;
    cfg.split_k = spec->split_k > 1 ? spec->split_k : 0; cfg.n_col_passes = 1; cfg.swap_grid = spec->swap_grid;
    cfg.wgp_mode = spec->wgp_mode;
    GemmCall g{};
    g.cfg = &cfg; g.trans_a = 0; g.trans_b = spec->transpose == T0B_TILE_NT; g.a = x; g.b = wt; g.c_dst[0] = y; g.n_dst = 1;
    g.m = m; g.n = n; g.k = k; g.lda = k; g.ldb = spec->transpose == T0B_TILE_NT ? k : n; g.ldc = n;
    g.out_bf16 = 0;
    rc = make_chain(ctx, spec->epilogue, static_cast<int32_t>(spec->n_epilogue), bias, scale, clamp_min, clamp_max, &g.epi);
    if (rc != T0B_OK) return rc;
    rc = run_gemm(ctx, g);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "t0b_tile_dispatch", 0);
}

int32_t t0b_gemm_time(t0b_ctx* ctx, const t0b_gemm_config* cfg, int32_t trans_a, int32_t trans_b, uint64_t a, uint64_t b,
                      uint64_t c, uint32_t m, uint32_t n, uint32_t k, uint64_t lda, uint64_t ldb, uint64_t ldc,
                      int32_t out_dtype, int32_t warmup, int32_t iters, float* ms) {
    int32_t rc = precheck(ctx);
    if (rc != T0B_OK) return rc;
    if (!ms || iters < 1) return set_error(ctx, T0B_ERR_INVALID, "gemm_time: bad arguments");
    for (int i = 0; i < warmup; ++i) {
        rc = t0b_gemm(ctx, cfg, trans_a, trans_b, a, b, c, m, n, k, lda, ldb, ldc, out_dtype, 0, 0, 1.0f, 0, 0, 1);
        if (rc != T0B_OK) return rc;
    }
    cudaEvent_t e0, e1;
    cudaEventCreate(&e0);
    cudaEventCreate(&e1);
    cudaStreamSynchronize(ctx->stream);
    cudaEventRecord(e0, ctx->stream);
    for (int i = 0; i < iters; ++i) {
        rc = t0b_gemm(ctx, cfg, trans_a, trans_b, a, b, c, m, n, k, lda, ldb, ldc, out_dtype, 0, 0, 1.0f, 0, 0, 1);
        if (rc != T0B_OK) break;
    }
    cudaEventRecord(e1, ctx->stream);
    cudaError_t e = cudaEventSynchronize(e1);
    float total = 0.0f;
    if (e == cudaSuccess) cudaEventElapsedTime(&total, e0, e1);
    cudaEventDestroy(e0);
    cudaEventDestroy(e1);
    if (rc != T0B_OK) return rc;
    if (e != cudaSuccess) return check_cuda(ctx, e, "gemm_time");
    const int st = take_device_status(ctx);
    if (st != 0) return set_error(ctx, T0B_ERR_DEVICE, "gemm_time: device status %d", st);
    *ms = total / static_cast<float>(iters);
    return T0B_OK;
}

int32_t t0b_tune(t0b_ctx* ctx, uint32_t m, uint32_t n, uint32_t k, int32_t trans_a, int32_t trans_b, int32_t out_dtype,
                 t0b_gemm_config* best, float* best_tflops) {
    int32_t rc = precheck(ctx);
    if (rc != T0B_OK) return rc;
    if (!best || m == 0 || n == 0 || k == 0) return set_error(ctx, T0B_ERR_INVALID, "tune: bad arguments");
    if (!ctx->autotune_dir.empty() && !trans_a && trans_b && out_dtype == T0B_OUT_F32) {
        // The disk cache is keyed by (M, N, K) only, like the reference's; it describes the NT / f32-out kernel.
        float tf = 0.0f;
        if (t0b_tune_cache_load(ctx->autotune_dir.c_str(), m, n, k, best, &tf) == T0B_OK) {
            if (best_tflops) *best_tflops = tf;
            tuned_remember(m, n, k, trans_a, trans_b, out_dtype == T0B_OUT_BF16, *best);
            return T0B_OK;
        }
    }
    const size_t elem = out_dtype == T0B_OUT_BF16 ? 2 : 4;
    uint64_t a = 0, b = 0, c = 0;
    rc = t0b_alloc(ctx, static_cast<size_t>(m) * k * 2, &a);
    if (rc == T0B_OK) rc = t0b_alloc(ctx, static_cast<size_t>(n) * k * 2, &b);
    if (rc == T0B_OK) rc = t0b_alloc(ctx, static_cast<size_t>(m) * n * elem, &c);
    const uint64_t lda = trans_a ? m : k, ldb = trans_b ? k : n;
    float best_ms = 1e30f;
    std::vector<std::pair<float, t0b_gemm_config>> survey;
    if (rc != T0B_OK) goto done;
    {
        const float scale = 1.7f / sqrtf(static_cast<float>(k));   // unit-variance-like products, as in the benchmark inputs
        fill_random_bf16_kernel<<<ctx->num_sms * 8, 256, 0, ctx->stream>>>(reinterpret_cast<__nv_bfloat16*>(a), static_cast<size_t>(m) * k, 0x1234u, scale);
        fill_random_bf16_kernel<<<ctx->num_sms * 8, 256, 0, ctx->stream>>>(reinterpret_cast<__nv_bfloat16*>(b), static_cast<size_t>(n) * k, 0x5678u, scale);
        rc = check_cuda(ctx, cudaGetLastError(), "tuner fill");
        if (rc != T0B_OK) goto done;
    }
    static const char* tiles[] = {"b200_256x512", "b200_512x256", "b200_256x256", "b200_256x128", "b200_128x256", "b200_128x128", "b200_128x64"};
    // Pass 1 surveys every candidate with a few launches.  Such a short measurement is noisy (clock ramps, power state),
    // so pass 2 re-times the best few of them, and the cost model's choice, with longer interleaved rounds and keeps
    // the best of that pass; the model's choice is only given up for something measurably faster.
    for (const char* t : tiles) {
        const uint32_t kb_total = (k + 63) / 64;
        for (uint32_t sk = 1; sk <= 16; sk *= 2) {
            if (sk > 1 && kb_total / sk < 2) break;
            t0b_gemm_config cfg;
            t0b_config_preset(t, &cfg);
            cfg.split_k = sk > 1 ? sk : 0;
            t0b_gemm_plan plan;
            PlanInput pin{m, n, k, trans_a, trans_b, lda, ldb, a, b, ctx->num_sms};
            resolve_plan(&cfg, pin, &plan);
            const uint64_t work = static_cast<uint64_t>((m + plan.bm - 1) / plan.bm) * ((n + plan.bn - 1) / plan.bn);
            if (sk > 1 && work * (sk / 2) >= static_cast<uint64_t>(ctx->num_sms) / plan.cta_group) break;   // already full
            // Rasterisation: both directions, and for tile counts of several waves a few group widths besides the
            // automatic one (0): narrow, medium, and the whole grouped dimension.
            static const uint32_t groups[] = {0, 2, 12, 4096};
            const int n_groups = work >= 2 * (static_cast<uint64_t>(ctx->num_sms) / plan.cta_group) ? 4 : 1;
            for (int gi = 0; gi < n_groups; ++gi) {
                for (uint32_t swap = 0; swap < 2; ++swap) {
                    cfg.swap_grid = swap;
                    cfg.lds_pad = groups[gi];
                    float ms = 0.0f;
                    rc = t0b_gemm_time(ctx, &cfg, trans_a, trans_b, a, b, c, m, n, k, lda, ldb, n, out_dtype, 2, 5, &ms);
                    if (rc != T0B_OK) goto done;
                    survey.emplace_back(ms, cfg);
                }
            }
        }
    }
    {
        std::sort(survey.begin(), survey.end(), [](const std::pair<float, t0b_gemm_config>& x, const std::pair<float, t0b_gemm_config>& y) { return x.first < y.first; });
        std::vector<t0b_gemm_config> finalists;
        t0b_gemm_config model;
        default_b200_config(m, k, n, ctx->num_sms, &model);
        finalists.push_back(model);
        for (size_t i = 0; i < survey.size() && finalists.size() < 4; ++i) finalists.push_back(survey[i].second);
        const float est = survey.empty() ? 1.0f : survey[0].first;
        const int iters = std::max(5, std::min(40, static_cast<int>(20.0f / std::max(est, 1e-3f))));   // about 20 ms per round
        std::vector<float> score(finalists.size(), 1e30f);
        for (int round = 0; round < 3; ++round) {
            for (size_t i = 0; i < finalists.size(); ++i) {
                float ms = 0.0f;
                rc = t0b_gemm_time(ctx, &finalists[i], trans_a, trans_b, a, b, c, m, n, k, lda, ldb, n, out_dtype, 1, iters, &ms);
                if (rc != T0B_OK) goto done;
                score[i] = std::min(score[i], ms);
            }
        }
        size_t pick = 0;   // the model's choice, unless another finalist is at least 1 % faster
        for (size_t i = 1; i < finalists.size(); ++i)
            if (score[i] < score[pick] * (pick == 0 ? 0.99f : 1.0f)) pick = i;
        best_ms = score[pick];
        *best = finalists[pick];
    }
done:
    // Every exit path returns the operands to the pool (only the ones that were obtained).
    if (a) t0b_recycle(ctx, a);
    if (b) t0b_recycle(ctx, b);
    if (c) t0b_recycle(ctx, c);
    if (rc != T0B_OK) return rc;
    const float tflops = 2.0f * m * n * static_cast<float>(k) / (best_ms * 1e-3f) / 1e12f;
    if (best_tflops) *best_tflops = tflops;
    tuned_remember(m, n, k, trans_a, trans_b, out_dtype == T0B_OUT_BF16, *best);   // config-less GEMM calls and t0b_auto_select answer from it
    if (!ctx->autotune_dir.empty() && !trans_a && trans_b && out_dtype == T0B_OUT_F32)
        t0b_tune_cache_save(ctx->autotune_dir.c_str(), m, n, k, best, best_tflops ? *best_tflops : 0.0f);
    return T0B_OK;
}

int32_t t0b_selftest_bounded_wait(t0b_ctx* ctx, uint64_t limit_ns) {
    int32_t rc = precheck(ctx);
    if (rc != T0B_OK) return rc;
    if (limit_ns == 0 || limit_ns > 5000000000ull) return set_error(ctx, T0B_ERR_INVALID, "selftest: limit must be in (0, 5e9] ns");
    bounded_wait_selftest_kernel<<<1, 32, 0, ctx->stream>>>(ctx->status_dev, limit_ns);
    rc = finish(ctx, 0, "bounded-wait self test");
    return rc;
}

}  // extern "C"
