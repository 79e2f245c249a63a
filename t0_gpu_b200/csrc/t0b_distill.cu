// Distillation from a teacher's top logits, on given student logits:
//   q = softmax over the row's teacher words of t_k / T                 (the teacher, over the words it gave)
//   p = softmax over the vocabulary of z_v / T                          (the student)
//   loss = sum_k q_k (log q_k - log p_{id_k})                           (Kullback-Leibler divergence)
//   d loss / d z_v = (p_v - sum_{k: id_k = v} q_k) / T
// Loss and gradient come from one read of the logits.  A row is shared by a thread-block cluster of 1 to 8 CTAs; each keeps
// its slice of the row in shared memory while it gathers the running maximum and sum, the CTAs exchange those two numbers
// over distributed shared memory, and the gradient is written from the cached slice.  HBM traffic: one read of z, one
// write of dz.  All statistics are f32.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "ptx_sm100.cuh"
#include "t0b_internal.hpp"

using namespace t0b;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kNoWord = 0xffffffffu;
constexpr int kMaxCluster = 8;
constexpr size_t kCacheMax = 200 * 1024;   // per CTA; a longer slice is read twice instead

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Block-wide sum / maximum; every thread receives it.  `red` holds kWarps floats.
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) t += red[i];
    return t;
}
__device__ __forceinline__ float block_max(float v, float* red) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = red[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) t = fmaxf(t, red[i]);
    return t;
}
// (m, s) <- the statistics of both halves: s = sum of 2^((z - m) c).  A half without any z above -inf has m = -inf, s = 0.
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2, float c) {
    const float mm = fmaxf(m, m2);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    s = s * exp2_approx((m - ref) * c) + s2 * exp2_approx((m2 - ref) * c);
    m = mm;
}

// 16 bytes of logits as floats.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
        v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_as(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// kN consecutive gradients, whole group in the row.
template <int N>
__device__ __forceinline__ void store_group(float* p, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) __stcs(reinterpret_cast<float4*>(p + i), make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
}
__device__ __forceinline__ void store_group(__nv_bfloat16* p, const float (&v)[8]) { __stcs(reinterpret_cast<uint4*>(p), Vec<__nv_bfloat16>::pack(v)); }
__device__ __forceinline__ void store_group(__nv_bfloat16* p, const float (&v)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)));
}

struct DistillParams {
    const void* logits;
    void* dlogits;
    const uint32_t* ids;
    const float* teacher;
    const float* weights;
    float* losses;
    uint32_t cols, topk;
    unsigned long long ld, ldk;
    float c, inv_t;          // log2(e) / T and 1 / T
    float scale;             // of the gradient, 1 / T included
    uint32_t groups_per_cta; // 16-byte groups of one CTA's slice
    int in_vec, out_vec;     // base pointers allow whole-group accesses
    int* status;
};

template <typename IN, typename OUT, bool CACHE>
__global__ void __launch_bounds__(kThreads) topk_distill_kernel(const DistillParams p) {
    constexpr int N = Vec<IN>::kN;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float red[kWarps];
    __shared__ float2 red2[kWarps];
    __shared__ __align__(16) float2 xch[kMaxCluster];
    uint4* cache = reinterpret_cast<uint4*>(smem);
    uint32_t* ids = reinterpret_cast<uint32_t*>(smem + (CACHE ? static_cast<size_t>(p.groups_per_cta) * 16 : 0));
    float* q = reinterpret_cast<float*>(ids + p.topk);
    uint32_t nranks, rank;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nranks));
    rank = ptx::cluster_ctarank();
    const uint32_t row = blockIdx.x / nranks;
    const int tid = threadIdx.x;
    ptx::cluster_arrive();   // every CTA of the cluster has started once the matching wait returns

    // The teacher's distribution; every CTA of the cluster computes all of it (at most 1024 words).
    float tmax = -INFINITY;
    for (uint32_t k = tid; k < p.topk; k += kThreads) {
        uint32_t id = p.ids[row * p.ldk + k];
        if (id != kNoWord && id >= p.cols) {
            if (rank == 0) *reinterpret_cast<volatile int*>(p.status) = kDevBadIndex;   // the word is left out
            id = kNoWord;
        }
        const float t = id == kNoWord ? -INFINITY : p.teacher[row * p.ldk + k];
        ids[k] = id;
        q[k] = t;
        tmax = fmaxf(tmax, t);
    }
    tmax = block_max(tmax, red);
    const float tref = tmax == -INFINITY ? 0.0f : tmax;
    float tsum = 0.0f;
    for (uint32_t k = tid; k < p.topk; k += kThreads) tsum += ids[k] == kNoWord ? 0.0f : expf((q[k] - tref) * p.inv_t);
    tsum = block_sum(tsum, red);
    const float tlog = logf(tsum);
    bool live = tsum > 0.0f || tsum != tsum;
    const IN* zr = static_cast<const IN*>(p.logits) + row * p.ld;
    float cross = 0.0f;   // rank 0: sum of q (log q - z / T) over this thread's words, z relative to the row's maximum later
    float qsum = 0.0f;
    const bool want_loss = rank == 0 && p.losses;
    constexpr int kOwn = 1024 / kThreads;   // words per thread at most
    float z_own[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const uint32_t k = tid + i * kThreads;
        z_own[i] = 0.0f;
        if (live && k < p.topk) {
            const float lq = (q[k] - tref) * p.inv_t - tlog;
            const float qk = ids[k] == kNoWord ? 0.0f : expf(lq);
            if (ids[k] != kNoWord) z_own[i] = to_float(zr[ids[k]]);   // before anything is written: dlogits may be the logits
            if (qk != 0.0f) cross += qk * lq;
            q[k] = qk;
        }
    }

    // This CTA's slice in 16-byte groups, counted from the 16-byte boundary at or before the row.
    const unsigned long long e0 = row * p.ld;
    const unsigned long long g0 = e0 / N;
    const uint32_t ngroups = static_cast<uint32_t>((e0 + p.cols - 1) / N - g0 + 1);
    const uint32_t lo = min(rank * p.groups_per_cta, ngroups), hi = min(lo + p.groups_per_cta, ngroups);
    const IN* zg = static_cast<const IN*>(p.logits) + g0 * N;
    const int lead = static_cast<int>(e0 - g0 * N);   // elements of group 0 that belong to the row before
    // Group g holds columns g * N - lead ...; read it whole, or element by element at the row's ends.
    auto load_group = [&](uint32_t g) -> uint4 {
        const long long col = static_cast<long long>(g) * N - lead;
        if (p.in_vec && col >= 0 && col + N <= p.cols) return __ldcs(reinterpret_cast<const uint4*>(zg) + g);
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (col + i >= 0 && col + i < p.cols) ? to_float(zr[col + i]) : -INFINITY;
        return Vec<IN>::pack(v);
    };
    float m = -INFINITY, s = 0.0f;
    if (live) {
        constexpr int U = 4;   // loads in flight per thread
        for (uint32_t g = lo + tid; g < hi; g += U * kThreads) {
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (g + u * kThreads < hi) raw[u] = load_group(g + u * kThreads);
            float lm = m;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (g + u * kThreads < hi) {
                    if (CACHE) cache[g + u * kThreads - lo] = raw[u];
                    float v[N];
                    Vec<IN>::unpack(raw[u], v);
#pragma unroll
                    for (int i = 0; i < N; ++i) lm = fmaxf(lm, v[i]);
                }
            const float ref = lm == -INFINITY ? 0.0f : lm;
            if (lm > m) s *= exp2_approx((m - ref) * p.c);
            m = lm;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (g + u * kThreads < hi) {
                    float v[N];
                    Vec<IN>::unpack(raw[u], v);
#pragma unroll
                    for (int i = 0; i < N; ++i) s += exp2_approx((v[i] - ref) * p.c);
                }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
            join_stats(m, s, m2, s2, p.c);
        }
        if ((tid & 31) == 0) red2[tid >> 5] = make_float2(m, s);
        __syncthreads();
        m = red2[0].x;
        s = red2[0].y;
#pragma unroll
        for (int i = 1; i < kWarps; ++i) join_stats(m, s, red2[i].x, red2[i].y, p.c);
    }
    // Exchange over the cluster: every CTA gets every (m, s) and joins them in rank order, so all hold the same bits.
    ptx::cluster_wait();
    if (tid < static_cast<int>(nranks)) {
        const uint32_t dst = ptx::mapa(ptx::smem_u32(&xch[rank]), static_cast<uint32_t>(tid));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(m), "f"(s) : "memory");
    }
    ptx::cluster_arrive();
    ptx::cluster_wait();
    m = xch[0].x;
    s = xch[0].y;
    for (uint32_t r = 1; r < nranks; ++r) join_stats(m, s, xch[r].x, xch[r].y, p.c);
    if (m == -INFINITY && s == 0.0f) live = false;   // every logit is -inf: the row has no distribution

    if (want_loss) {
        const float lse = logf(s);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const uint32_t k = tid + i * kThreads;
            if (live && k < p.topk && q[k] != 0.0f) {
                cross -= q[k] * ((z_own[i] - m) * p.inv_t);
                qsum += q[k];
            }
        }
        cross = block_sum(cross, red);
        qsum = block_sum(qsum, red);
        if (tid == 0) p.losses[row] = live ? cross + qsum * lse : 0.0f;
    }
    if (!p.dlogits) return;
    OUT* dr = static_cast<OUT*>(p.dlogits) + e0;
    OUT* dg = static_cast<OUT*>(p.dlogits) + g0 * N;
    const float a = live ? p.scale * (p.weights ? p.weights[row] : 1.0f) : 0.0f;
    const float inv = a / s;
    for (uint32_t g = lo + tid; g < hi; g += kThreads) {
        const long long col = static_cast<long long>(g) * N - lead;
        float v[N];
        if (live) {
            Vec<IN>::unpack(CACHE ? cache[g - lo] : load_group(g), v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = exp2_approx((v[i] - m) * p.c) * inv;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 0.0f;
        }
        if (p.out_vec && col >= 0 && col + N <= p.cols) {
            store_group(dg + static_cast<size_t>(g) * N, v);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col + i >= 0 && col + i < p.cols) store_as(dr + col + i, v[i]);
        }
    }
    if (!live) return;
    // The teacher's words of this slice, after their neighbours: one thread per distinct word writes p - (its q).
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const uint32_t k = tid + i * kThreads;
        if (k >= p.topk) break;
        const uint32_t id = ids[k];
        const uint32_t g = (id + lead) / N;
        if (id == kNoWord || g < lo || g >= hi) continue;
        bool first = true;
        for (uint32_t j = 0; j < k; ++j) first = first && ids[j] != id;
        if (!first) continue;
        float qk = q[k];
        for (uint32_t j = k + 1; j < p.topk; ++j)
            if (ids[j] == id) qk += q[j];
        store_as(dr + id, a * (exp2_approx((z_own[i] - m) * p.c) / s - qk));
    }
}

// Dynamic shared memory above 48 KB has to be asked for once per kernel and device.
template <typename IN, typename OUT, bool CACHE>
int32_t launch_distill(t0b_ctx* ctx, const DistillParams& p, uint32_t rows, uint32_t nranks, size_t smem) {
    auto kfn = topk_distill_kernel<IN, OUT, CACHE>;
    static std::atomic<bool> configured[64];
    std::atomic<bool>& done = configured[ctx->device & 63];
    if (!done.load(std::memory_order_acquire)) {
        const int32_t rc = check_cuda(ctx, cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kCacheMax + 8 * 1024 + 16)),
                                      "cudaFuncSetAttribute(topk_distill)");
        if (rc != T0B_OK) return rc;
        done.store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * nranks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return check_cuda(ctx, cudaLaunchKernelEx(&cfg, kfn, p), "cudaLaunchKernelEx(topk_distill)");
}

}  // namespace

extern "C" {

int32_t t0b_topk_distill(t0b_ctx* ctx, uint64_t logits, int32_t logits_dtype, uint64_t ids, uint64_t teacher, uint64_t row_weights,
                         uint64_t losses, uint64_t dlogits, int32_t grad_dtype, uint32_t rows, uint32_t cols, uint64_t ld,
                         uint32_t topk, uint64_t ldk, float temperature, float scale, int32_t async) {
    int32_t rc = precheck(ctx);
    if (rc != T0B_OK) return rc;
    if (rows == 0) return T0B_OK;
    if (logits_dtype != T0B_OUT_F32 && logits_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: unknown logits_dtype %d", logits_dtype);
    if (dlogits && grad_dtype != T0B_OUT_F32 && grad_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: unknown grad_dtype %d", grad_dtype);
    if (!logits || !ids || !teacher || (!losses && !dlogits)) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: null pointer");
    if (cols == 0 || cols > 0x7fffff00u || ld < cols) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: %u columns with a pitch of %llu", cols, static_cast<unsigned long long>(ld));
    if (topk == 0 || topk > T0B_MAX_TOPK || ldk < topk)
        return set_error(ctx, T0B_ERR_INVALID, "topk_distill: topk %u is outside 1..%d, or its pitch %llu is smaller", topk, T0B_MAX_TOPK, static_cast<unsigned long long>(ldk));
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(scale))
        return set_error(ctx, T0B_ERR_INVALID, "topk_distill: temperature %g must be positive and finite, scale %g finite", temperature, scale);
    const size_t ie = logits_dtype == T0B_OUT_BF16 ? 2 : 4, oe = grad_dtype == T0B_OUT_BF16 ? 2 : 4;
    if (logits % ie || (dlogits && dlogits % oe) || ids % 4 || teacher % 4 || losses % 4 || row_weights % 4)
        return set_error(ctx, T0B_ERR_INVALID, "topk_distill: a pointer is not aligned to its element");
    if (dlogits == logits && ie != oe) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: a gradient in the place of the logits needs their type");
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    rc = check_fits(ctx, "topk_distill", {{"logits", logits, ((rows - 1ull) * ld + cols) * ie}, {"dlogits", dlogits, ((rows - 1ull) * ld + cols) * oe},
                                          {"ids", ids, ((rows - 1ull) * ldk + topk) * 4}, {"teacher", teacher, ((rows - 1ull) * ldk + topk) * 4},
                                          {"losses", losses, rows * 4ull}, {"row_weights", row_weights, rows * 4ull}});
    if (rc != T0B_OK) return rc;

    const uint32_t n = static_cast<uint32_t>(16 / ie);
    DistillParams p{};
    p.logits = reinterpret_cast<const void*>(logits);
    p.dlogits = reinterpret_cast<void*>(dlogits);
    p.ids = reinterpret_cast<const uint32_t*>(ids);
    p.teacher = reinterpret_cast<const float*>(teacher);
    p.weights = reinterpret_cast<const float*>(row_weights);
    p.losses = reinterpret_cast<float*>(losses);
    p.cols = cols; p.topk = topk; p.ld = ld; p.ldk = ldk;
    p.inv_t = 1.0f / temperature;
    p.c = 1.4426950408889634f / temperature;
    p.scale = scale / temperature;
    p.in_vec = logits % 16 == 0;
    p.out_vec = dlogits % std::min<size_t>(16, n * oe) == 0;
    p.status = ctx->status_dev;
    // CTAs per row: enough that four slices fit an SM (their loads and stores overlap each other), and more while few rows
    // would leave SMs idle and the slices stay worth a CTA.
    const size_t groups = (static_cast<size_t>(cols) + n - 1) / n + 1;   // one more where rows start off a 16-byte boundary
    uint32_t nranks = 1;
    while (nranks < kMaxCluster && groups * 16 / nranks > 48 * 1024) nranks *= 2;
    while (nranks < kMaxCluster && static_cast<uint64_t>(rows) * nranks < static_cast<uint64_t>(ctx->num_sms) && groups * 16 / nranks >= 8 * 1024) nranks *= 2;
    if (static_cast<uint64_t>(rows) * nranks > 0x7fffffffull) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: %u rows are too many", rows);
    p.groups_per_cta = static_cast<uint32_t>((groups + nranks - 1) / nranks);
    const bool cached = p.groups_per_cta * 16ull <= kCacheMax;
    const size_t smem = (cached ? p.groups_per_cta * 16ull : 0) + topk * 8ull;
    const bool in16 = ie == 2, out16 = oe == 2;
    if (in16) {
        if (out16) rc = cached ? launch_distill<__nv_bfloat16, __nv_bfloat16, true>(ctx, p, rows, nranks, smem) : launch_distill<__nv_bfloat16, __nv_bfloat16, false>(ctx, p, rows, nranks, smem);
        else rc = cached ? launch_distill<__nv_bfloat16, float, true>(ctx, p, rows, nranks, smem) : launch_distill<__nv_bfloat16, float, false>(ctx, p, rows, nranks, smem);
    } else {
        if (out16) rc = cached ? launch_distill<float, __nv_bfloat16, true>(ctx, p, rows, nranks, smem) : launch_distill<float, __nv_bfloat16, false>(ctx, p, rows, nranks, smem);
        else rc = cached ? launch_distill<float, float, true>(ctx, p, rows, nranks, smem) : launch_distill<float, float, false>(ctx, p, rows, nranks, smem);
    }
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "topk_distill");
}

}  // extern "C"
