// Distillation from a teacher's top logits, on given student logits:
//   q = softmax over the row's teacher words of t_k / T                 (the teacher, over the words it gave)
//   p = softmax over the vocabulary of z_v / T                          (the student)
//   loss = sum_k q_k (log q_k - log p_{id_k})                           (Kullback-Leibler divergence)
//   d loss / d z_v = (p_v - sum_{k: id_k = v} q_k) / T
// HBM bounds the kernels: one read of z, one write of dz (streamed rows and the general form read z again, from L2 where it is
// still there: 644 MB for 2048 x 128000 bf16, of 524).  Three forms:
//   rows in registers  a cluster of 1 to 8 CTAs per row; every thread keeps up to sixteen 16-byte groups, all loaded before
//                      the first is used: maximum; exponentials, which replace the logits, and their sum; -- the CTAs
//                      exchange (maximum, sum) over distributed shared memory -- gradient = exponential times one factor
//   streamed rows      long rows, enough of them for every SM: one CTA per row, which L2 serves the second time
//   any rows           pointers off their 16-byte boundaries
// Rows in registers keep the exponentials of bf16 logits in 16 bits as fp16, 2^15 times what they are relative to their CTA's
// maximum (11 significant bits down to 2^-29 of it, at most 2^-40 of it off below), where the gradient is bf16 as well: making
// them again would cost 7 to 15 % (4096 x 32000: 155 us instead of 135 us).  For an f32 gradient they are computed again.
// Statistics, losses and the gradient at the teacher's words are f32 throughout.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_pipeline.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "ptx_sm100.cuh"
#include "t0b_internal.hpp"

using namespace t0b;

namespace {

constexpr int kThreads = 256;         // rows in registers, and the general form
constexpr uint32_t kNoWord = 0xffffffffu;
constexpr int kMaxCluster = 8;

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
// Block-wide maxima / sums of two values at once; every thread receives them.  `red` is used by one call only.
template <int T>
__device__ __forceinline__ void block_max2(float& a, float& b, float2* red) {
    a = warp_max(a);
    b = warp_max(b);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = red[0].x;
    b = red[0].y;
#pragma unroll
    for (int i = 1; i < T / 32; ++i) {
        a = fmaxf(a, red[i].x);
        b = fmaxf(b, red[i].y);
    }
}
template <int T>
__device__ __forceinline__ void block_sum2(float& a, float& b, float2* red) {
    a = warp_sum(a);
    b = warp_sum(b);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
        a += red[i].x;
        b += red[i].y;
    }
}

// exp(z / T) relative to the largest z of a set, as 2^(z c - mc) with c = log2(e) / T and mc = m c rounded: one fused
// multiply-add whose only rounding is that of the small difference, and references that subtract exactly from one another.
// The rounding of mc, up to |mc| 2^-24, is part of every exponent; up to |mc| = 2^22 that is a factor of at most 2^(1/4), which
// cancels.  Beyond (a row masked with -1e9 as a whole, logits at the type's lowest value) the difference is taken first.
struct Ref {
    float m, mc;
    bool fused;
    __device__ __forceinline__ Ref(float m_, float c) : m(m_), mc(m_ * c), fused(fabsf(m_ * c) <= 4194304.0f) {
        if (m_ == -INFINITY) { m = mc = 0.0f; fused = true; }   // nothing in the set: exponentials 0, not exp(-inf + inf)
    }
    __device__ __forceinline__ float arg(float z, float c) const { return fused ? fmaf(z, c, -mc) : (z - m) * c; }
    // (z - m) / T, as the exponent's counterpart in the loss.
    __device__ __forceinline__ float log_of(float z, float c, float inv_t) const { return fused ? 0.6931471805599453f * fmaf(z, c, -mc) : (z - m) * inv_t; }
    // What an exponential relative to this reference is worth relative to `other` (>= this one): 2 to the difference of the two
    // references, mc where a side is fused and m c, unrounded, where it is not.
    __device__ __forceinline__ float to(const Ref& other, float c) const {
        const float d = fused ? (other.fused ? mc - other.mc : fmaf(-other.m, c, mc)) : (other.fused ? fmaf(m, c, -other.mc) : (m - other.m) * c);
        return exp2_approx(d);
    }
};

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
    uint32_t table;          // slots of the words' hash table (2^(32 - table_shift)), 0: none
    uint32_t table_shift;
    uint32_t groups_per_cta; // 16-byte groups of one CTA's slice (rows in registers)
    int* status;
};

// v <- 2^(v c - mc), the exponentials relative to `r`.
template <int N>
__device__ __forceinline__ void exp_group(float (&v)[N], const Ref& r, float c) {
    if (r.fused) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = exp2_approx(fmaf(v[e], c, -r.mc));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = exp2_approx((v[e] - r.m) * c);
    }
}

// What the exponentials are kept as between the passes, kScale times what they are: f32 logits f32, bf16 logits fp16 -- an
// exponential is at most 2^(1/4) (Ref), so that the largest are below 2^15.25 and fit.
template <typename T> struct Kept;
template <> struct Kept<float> {
    static constexpr float kScale = 1.0f;
    static __device__ __forceinline__ uint4 pack(const float (&e)[4]) { return Vec<float>::pack(e); }
    static __device__ __forceinline__ void unpack(const uint4& q, float (&e)[4]) { Vec<float>::unpack(q, e); }
};
template <> struct Kept<__nv_bfloat16> {
    static constexpr float kScale = 32768.0f;
    static __device__ __forceinline__ uint4 pack(const float (&e)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(kScale * e[2 * i], kScale * e[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void unpack(const uint4& q, float (&e)[8]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            e[2 * i] = f.x;
            e[2 * i + 1] = f.y;
        }
    }
};

// Maximum of a group, NaN left out (it shows in the sum).
__device__ __forceinline__ float group_max(const uint4& q, const float*) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
}
__device__ __forceinline__ float group_max(const uint4& q, const __nv_bfloat16*) {
    auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(h(q.x), h(q.y)), __hmax2(h(q.z), h(q.w)));
    return fmaxf(__low2float(m), __high2float(m));
}

// The teacher's side of a row in one CTA of T threads: each owns the words tid, tid + T, ..., kOwn of them at most (one,
// where the call's topk allows it: three registers a word).
template <int T, int kOwn>
struct Words {
    uint32_t id[kOwn];
    float t[kOwn], z[kOwn];   // t: the teacher's logit, then q
    float tmax;

    // A hash table of the row's words (`size` slots, a power of two, at least twice the words; kNoWord = free) finds out
    // whether a word is named twice: clear() before one block-wide barrier, mark() behind it, `twice` is valid behind the
    // next.  Without slots every row counts as one with a word named twice.
    static __device__ __forceinline__ void clear(uint32_t* table, uint32_t size, int* twice) {
        for (uint32_t i = threadIdx.x; i < size; i += T) table[i] = kNoWord;
        if (threadIdx.x == 0) *twice = size == 0;
    }
    __device__ __forceinline__ void mark(const DistillParams& p, uint32_t* table, uint32_t size, int* twice) const {
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (mine(p, i) && id[i] != kNoWord) {
                // 2^32 / the golden ratio; the product's high bits, which every bit of the id reaches: ids with the same low
                // bits (any stride of a power of two) spread as well (2000 x 16000 f32, 31 words 512 apart: 61 us, as for random
                // words; 270 us with the low bits).
                uint32_t at = (id[i] * 2654435769u) >> p.table_shift;
                uint32_t old;
                while ((old = atomicCAS(table + at, kNoWord, id[i])) != kNoWord) {   // ends: at most half of the slots are taken
                    if (old == id[i]) {
                        *twice = 1;
                        break;
                    }
                    at = (at + 1) & (size - 1);
                }
            }
    }

    // Warps beyond the last word skip all of it.
    static __device__ __forceinline__ bool mine(const DistillParams& p, int i) { return i * T + (threadIdx.x & ~31u) < p.topk; }

    template <typename IN>
    __device__ __forceinline__ void load(const DistillParams& p, uint32_t row, const IN* zr, bool report) {
        tmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            id[i] = kNoWord;
            t[i] = z[i] = 0.0f;
            const uint32_t k = threadIdx.x + i * T;
            if (mine(p, i) && k < p.topk) {
                id[i] = p.ids[row * p.ldk + k];
                t[i] = p.teacher[row * p.ldk + k];
            }
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (mine(p, i)) {
                if (id[i] != kNoWord && id[i] >= p.cols) {
                    if (report) *reinterpret_cast<volatile int*>(p.status) = kDevBadIndex;   // the word is left out
                    id[i] = kNoWord;
                }
                if (id[i] != kNoWord) {
                    z[i] = to_float(zr[id[i]]);   // before anything is written: dlogits may be the logits
                    tmax = fmaxf(tmax, t[i]);
                }
            }
    }
    // Sum of exp((t - max) / T) over this thread's words.
    __device__ __forceinline__ float sum(const DistillParams& p, float tref) const {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (mine(p, i) && id[i] != kNoWord) s += expf((t[i] - tref) * p.inv_t);
        return s;
    }
    // t becomes q; ids and q go to shared memory; returns sum q log q and sum q over this thread's words.
    __device__ __forceinline__ float2 probs(const DistillParams& p, float tref, float tsum, bool live, uint32_t* sh_ids, float* sh_q) {
        float cross = 0.0f, qsum = 0.0f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (mine(p, i)) {
                const uint32_t k = threadIdx.x + i * T;
                const float lq = (t[i] - tref) * p.inv_t - logf(tsum);
                const float qk = (live && id[i] != kNoWord) ? expf(lq) : 0.0f;
                if (qk != 0.0f) {
                    cross += qk * lq;
                    qsum += qk;
                }
                t[i] = qk;
                if (k < p.topk) {
                    sh_ids[k] = id[i];
                    sh_q[k] = qk;
                }
            }
        return make_float2(cross, qsum);
    }
    // - sum q (z - m) / T over this thread's words.
    __device__ __forceinline__ float cross(const DistillParams& p, const Ref& all) const {
        float c = 0.0f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (mine(p, i) && t[i] != 0.0f) c -= t[i] * all.log_of(z[i], p.c, p.inv_t);
        return c;
    }
    // The gradient at the words of columns [c_lo, c_hi): one thread per distinct word writes a (p - its q).  Only where a word
    // may be named twice do the threads look through all of them.
    template <typename OUT>
    __device__ __forceinline__ void gradient(const DistillParams& p, const Ref& all, float a, float total, long long c_lo, long long c_hi,
                                             const uint32_t* sh_ids, const float* sh_q, bool twice, OUT* dr) const {
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (mine(p, i) && id[i] != kNoWord && id[i] >= c_lo && id[i] < c_hi) {
                const uint32_t k = threadIdx.x + i * T;
                float qk = t[i];
                if (twice) {
                    bool first = true;
                    for (uint32_t j = 0; j < k; ++j) first = first && sh_ids[j] != id[i];
                    if (!first) continue;
                    for (uint32_t j = k + 1; j < p.topk; ++j)
                        if (sh_ids[j] == id[i]) qk += sh_q[j];
                }
                store_as(dr + id[i], a * (exp2_approx(all.arg(z[i], p.c)) / total - qk));
            }
    }
};

struct RowStats { float m, total; };

// Every CTA of the cluster gets every CTA's (m, s) and joins them in rank order, so all hold the same bits.  `between` runs
// while the exchange is under way.
template <typename F>
__device__ __forceinline__ RowStats exchange(float m, float s, float c, uint32_t nranks, uint32_t rank, float2* xch, F&& between) {
    if (nranks == 1) {
        between();
        return {m, s};
    }
    ptx::cluster_wait();   // every CTA has started
    if (threadIdx.x < nranks) {
        const uint32_t dst = ptx::mapa(ptx::smem_u32(&xch[rank]), threadIdx.x);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(m), "f"(s) : "memory");
    }
    ptx::cluster_arrive();
    between();
    ptx::cluster_wait();
    RowStats st{xch[0].x, 0.0f};
    for (uint32_t r = 1; r < nranks; ++r) st.m = fmaxf(st.m, xch[r].x);
    const Ref all(st.m, c);
    for (uint32_t r = 0; r < nranks; ++r) st.total += xch[r].x == -INFINITY ? xch[r].y : xch[r].y * Ref(xch[r].x, c).to(all, c);
    return st;
}

// Where a row's whole 16-byte groups are: `front` columns before the first, `groups` of them, `back` columns behind the last.
template <typename IN>
struct RowSpan {
    unsigned long long e0, g_first;
    uint32_t front, groups, back;
    __device__ __forceinline__ RowSpan(const DistillParams& p, uint32_t row) {
        constexpr int N = Vec<IN>::kN;
        e0 = row * p.ld;
        g_first = (e0 + N - 1) / N;
        const unsigned long long g_end = (e0 + p.cols) / N;
        groups = g_end > g_first ? static_cast<uint32_t>(g_end - g_first) : 0;
        front = min(p.cols, static_cast<uint32_t>(g_first * N - e0));   // a row within one or two groups may have no whole one
        back = p.cols - front - groups * N;
    }
    __device__ __forceinline__ const uint4* at(const DistillParams& p) const {
        return reinterpret_cast<const uint4*>(static_cast<const IN*>(p.logits) + g_first * Vec<IN>::kN);
    }
};

// The columns of one of the row's ends as a group, filled up with -inf.
template <typename IN>
__device__ __forceinline__ uint4 edge_group(const DistillParams& p, const RowSpan<IN>& span, bool at_back) {
    constexpr int N = Vec<IN>::kN;
    const IN* z = static_cast<const IN*>(p.logits) + span.e0 + (at_back ? p.cols - span.back : 0);
    const uint32_t count = at_back ? span.back : span.front;
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < count ? to_float(z[e]) : -INFINITY;
    return Vec<IN>::pack(v);
}

// Rows of more than 64 KB, at least one for every SM: one CTA per row, two an SM.  The row is streamed twice, for the
// statistics and for the gradient.  Each thread's 16-byte groups arrive in batches through its own slots of a ring in shared
// memory, asked for two batches ahead; the last three batches are still there for the second pass, the others come from L2
// or, where the rows under way (76 MB of a 128000-word bf16 batch) have pushed them out, from HBM again.
// On one B200, 4096 x 128000 bf16 with gradient: 430 us (2.1 GB read and written once, 4.9 TB/s; HBM moves more with what
// comes twice), 455 us with the ring through both passes, 560 us with clusters that keep fewer rows under way, 640 us with the
// row in the registers of a cluster.  2048 x 50257 f32, losses alone: 75 us (5.5 TB/s).
constexpr int kStreamThreads = 512, kRingBatch = 4, kRingBatches = 3;
template <typename IN, typename OUT, int OWN>
__global__ void __launch_bounds__(kStreamThreads, 2) topk_distill_stream_kernel(const DistillParams p) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    constexpr int N = Vec<IN>::kN, T = kStreamThreads, B = kRingBatch, S = kRingBatches;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 red_max[T / 32], red_sum[T / 32], red_loss[T / 32];
    uint4* ring = reinterpret_cast<uint4*>(smem);        // slot j of thread t: ring[j * T + t]
    uint32_t* ids = reinterpret_cast<uint32_t*>(smem + static_cast<size_t>(B) * S * T * 16);
    float* q = reinterpret_cast<float*>(ids + p.topk);
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const RowSpan<IN> span(p, row);
    const IN* zr = static_cast<const IN*>(p.logits) + span.e0;
    const uint4* zg = span.at(p);
    const uint32_t batches = (span.groups + T * B - 1) / (T * B);
    // Batch n goes to ring batch n % S; always one group of copies, empty or not, so that "all but the last S - 1 groups" is
    // the batch in turn.
    auto ask = [&](uint32_t n) {
        if (n < batches) {
            const uint32_t first = n * (B * T) + tid;
            const uint32_t slot = (n % S) * B;
#pragma unroll
            for (int u = 0; u < B; ++u)
                if (first + u * T < span.groups) __pipeline_memcpy_async(ring + (slot + u) * T + tid, zg + first + u * T, 16);
        }
        __pipeline_commit();
    };
#pragma unroll
    for (int n = 0; n < S - 1; ++n) ask(n);
    Words<T, OWN> words;
    words.load(p, row, zr, true);

    // This thread's running maximum and sum.
    const IN* kind = nullptr;
    float m = -INFINITY, s = 0.0f;
    Ref cur(m, p.c);
    auto add = [&](const uint4 (&raw)[B], const bool (&have)[B]) {
        float lm = m;
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (have[u]) lm = fmaxf(lm, group_max(raw[u], kind));
        if (lm > m) {
            const Ref next(lm, p.c);
            if (m != -INFINITY) s *= cur.to(next, p.c);
            m = lm;
            cur = next;
        }
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (have[u]) {
                float v[N];
                Vec<IN>::unpack(raw[u], v);
                exp_group(v, cur, p.c);
#pragma unroll
                for (int e = 0; e < N; e += 4) s += (v[e] + v[e + 1]) + (v[e + 2] + v[e + 3]);
            }
    };
    for (uint32_t n = 0; n < batches; ++n) {
        ask(n + S - 1);
        __pipeline_wait_prior(S - 1);   // a thread reads only what it asked for itself
        const uint32_t first = n * (B * T) + tid, slot = (n % S) * B;
        uint4 raw[B];
        bool have[B];
#pragma unroll
        for (int u = 0; u < B; ++u) {
            have[u] = first + u * T < span.groups;
            raw[u] = have[u] ? ring[(slot + u) * T + tid] : make_uint4(0, 0, 0, 0);
        }
        add(raw, have);
    }
    // The columns outside whole groups, at most N - 1 at each end: one thread each.
    if (tid < 2) {
        uint4 raw[B];
        const bool have[B] = {true, false, false, false};
        raw[0] = edge_group<IN>(p, span, tid != 0);
        add(raw, have);
    }
    float mall = m;
    block_max2<T>(mall, words.tmax, red_max);
    const Ref all(mall, p.c);
    if (m != -INFINITY) s *= cur.to(all, p.c);
    const float tref = words.tmax == -INFINITY ? 0.0f : words.tmax;
    float tsum = words.sum(p, tref);
    block_sum2<T>(s, tsum, red_sum);
    bool live = tsum > 0.0f || tsum != tsum;
    float2 cq = words.probs(p, tref, tsum, live, ids, q);
    if (mall == -INFINITY && s == 0.0f) live = false;   // every logit is -inf: the row has no distribution
    if (p.losses) {
        if (live) cq.x += words.cross(p, all);
        block_sum2<T>(cq.x, cq.y, red_loss);
        if (tid == 0) p.losses[row] = live ? fmaf(cq.y, logf(s), cq.x) : 0.0f;
    }
    if (!p.dlogits) return;
    OUT* dr = static_cast<OUT*>(p.dlogits) + span.e0;
    OUT* dg = static_cast<OUT*>(p.dlogits) + span.g_first * N;
    const float a = live ? p.scale * (p.weights ? p.weights[row] : 1.0f) : 0.0f;
    const float inv = a / s;
    auto gradient = [&](const uint4& g, float (&v)[N]) {
        Vec<IN>::unpack(g, v);
        if (live) exp_group(v, all, p.c);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = live ? v[e] * inv : 0.0f;
    };
    // The columns outside whole groups first: with dlogits in the place of the logits they are read here once more.
    if (tid < 2) {
        float v[N];
        gradient(edge_group<IN>(p, span, tid != 0), v);
        const uint32_t col = tid == 0 ? 0 : p.cols - span.back, count = tid == 0 ? span.front : span.back;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < count) store_as(dr + col + e, v[e]);
    }
    // In place, too, a thread reads and writes its own groups only.  The last S batches are still in the ring; the reads of
    // the others let go of their lines in L2, and the next batch is under way while one is used.
    const uint32_t from_l2 = batches > S ? batches - S : 0;
    uint4 next[B];
    auto fetch = [&](uint32_t n) {
#pragma unroll
        for (int u = 0; u < B; ++u) {
            const uint32_t i = n * (B * T) + u * T + tid;
            if (n < from_l2) next[u] = __ldcs(zg + i);   // a batch with others behind it is whole
            else if (i < span.groups) next[u] = ring[((n % S) * B + u) * T + tid];
        }
    };
    fetch(0);
    for (uint32_t n = 0; n < batches; ++n) {
        uint4 raw[B];
#pragma unroll
        for (int u = 0; u < B; ++u) raw[u] = next[u];
        fetch(n + 1);
        const uint32_t first = n * (B * T) + tid;
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (first + u * T < span.groups) {
                float v[N];
                gradient(raw[u], v);
                store_group(dg + static_cast<size_t>(first + u * T) * N, v);
            }
    }
    __syncthreads();   // the words after their neighbours
    if (live) words.gradient(p, all, a, s, 0, p.cols, ids, q, true, dr);
}

// The fast form: base pointers on 16-byte boundaries (any pitch).  A row's whole
// 16-byte groups are divided among the cluster's threads, G to each at most, and the partial groups at its two ends go to
// one thread each (an extra group that only their warps look at).
template <typename IN, typename OUT, int G, int T, int OWN>
__global__ void __launch_bounds__(T, (G == 16 ? 2 : (G == 8 ? 3 : 4)) * 256 / T) topk_distill_kernel(const DistillParams p) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    constexpr int N = Vec<IN>::kN;
    constexpr bool kKeepExp = !(sizeof(IN) == 2 && sizeof(OUT) == 4);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 red_max[T / 32], red_sum[T / 32], red_loss[T / 32];
    __shared__ __align__(16) float2 xch[kMaxCluster];
    uint32_t* ids = reinterpret_cast<uint32_t*>(smem);
    float* q = reinterpret_cast<float*>(ids + p.topk);
    uint32_t* table = reinterpret_cast<uint32_t*>(q + p.topk);
    __shared__ int twice;
    uint32_t nranks;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nranks));
    const uint32_t rank = ptx::cluster_ctarank();
    const uint32_t row = blockIdx.x / nranks;
    const uint32_t tid = threadIdx.x;
    if (nranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;");

    const RowSpan<IN> span(p, row);
    const uint32_t lo = min(rank * p.groups_per_cta, span.groups), n_own = min(p.groups_per_cta, span.groups - lo);
    const IN* zr = static_cast<const IN*>(p.logits) + span.e0;
    const uint4* zg = span.at(p) + lo;
    const bool at_back = tid != 0;
    const bool has_edge = (tid == 0 && rank == 0 && span.front > 0) || (tid == 32 && rank == nranks - 1 && span.back > 0);

    uint4 raw[G];
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (tid + i * T < n_own) raw[i] = __ldcs(zg + tid + i * T);
    uint4 edge = make_uint4(0, 0, 0, 0);
    if (has_edge) edge = edge_group<IN>(p, span, at_back);
    Words<T, OWN> words;
    words.load(p, row, zr, rank == 0);
    words.clear(table, p.table, &twice);

    // Maximum of the slice (and of the teacher's logits), over the CTA.
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (tid + i * T < n_own) m = fmaxf(m, group_max(raw[i], static_cast<const IN*>(nullptr)));
    if (has_edge) m = fmaxf(m, group_max(edge, static_cast<const IN*>(nullptr)));
    block_max2<T>(m, words.tmax, red_max);
    if (p.table) words.mark(p, table, p.table, &twice);
    // Exponentials relative to it, and their sum.
    const Ref own(m, p.c);
    const bool nothing = m == -INFINITY;   // in this slice
    float s = 0.0f;
    auto exponentials = [&](uint4& g, bool fused) {
        float v[N];
        Vec<IN>::unpack(g, v);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = exp2_approx(fused ? fmaf(v[e], p.c, -own.mc) : (v[e] - own.m) * p.c);
#pragma unroll
        for (int e = 0; e < N; e += 4) s += (v[e] + v[e + 1]) + (v[e + 2] + v[e + 3]);
        if (kKeepExp) g = Kept<IN>::pack(v);
    };
    if (own.fused) {
#pragma unroll
        for (int i = 0; i < G; ++i)
            if (tid + i * T < n_own) exponentials(raw[i], true);
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i)
            if (tid + i * T < n_own) exponentials(raw[i], false);
    }
    if (has_edge) exponentials(edge, own.fused);
    const float tref = words.tmax == -INFINITY ? 0.0f : words.tmax;
    float tsum = words.sum(p, tref);
    block_sum2<T>(s, tsum, red_sum);
    bool live = tsum > 0.0f || tsum != tsum;
    float2 cq;
    const RowStats st = exchange(m, s, p.c, nranks, rank, xch, [&] { cq = words.probs(p, tref, tsum, live, ids, q); });
    const Ref all(st.m, p.c);
    if (st.m == -INFINITY && st.total == 0.0f) live = false;   // every logit is -inf: the row has no distribution
    if (rank == 0 && p.losses) {
        if (live) cq.x += words.cross(p, all);
        block_sum2<T>(cq.x, cq.y, red_loss);
        if (tid == 0) p.losses[row] = live ? fmaf(cq.y, logf(st.total), cq.x) : 0.0f;
    }
    if (!p.dlogits) return;
    OUT* dr = static_cast<OUT*>(p.dlogits) + span.e0;
    OUT* dg = static_cast<OUT*>(p.dlogits) + (span.g_first + lo) * N;
    const float a = live ? p.scale * (p.weights ? p.weights[row] : 1.0f) : 0.0f;
    const float inv = a / st.total;
    const float f = kKeepExp ? (nothing ? 0.0f : own.to(all, p.c) * inv * (1.0f / Kept<IN>::kScale)) : inv;
    auto gradient = [&](const uint4& g, float (&v)[N]) {
        if (kKeepExp) {
            Kept<IN>::unpack(g, v);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = live ? v[e] * f : 0.0f;
        } else {
            Vec<IN>::unpack(g, v);
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = live ? exp2_approx(all.arg(v[e], p.c)) * f : 0.0f;
        }
    };
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (tid + i * T < n_own) {
            float v[N];
            gradient(raw[i], v);
            store_group(dg + static_cast<size_t>(tid + i * T) * N, v);
        }
    if (has_edge) {
        float v[N];
        gradient(edge, v);
        const uint32_t col = at_back ? p.cols - span.back : 0, count = at_back ? span.back : span.front;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < count) store_as(dr + col + e, v[e]);
    }
    if (!live) return;
    __syncthreads();   // the words after their neighbours
    const long long c_lo = (rank == 0 ? 0 : static_cast<long long>(span.front) + static_cast<long long>(lo) * N);
    const long long c_hi = (rank == nranks - 1 ? p.cols : static_cast<long long>(span.front) + static_cast<long long>(lo + n_own) * N);
    words.gradient(p, all, a, st.total, c_lo, c_hi, ids, q, twice != 0, dr);
}

// The general form, one CTA per row: base pointers off their 16-byte boundaries, or rows longer than a cluster's registers.
// Every pass reads the row by element again (from L2, where it fits).
template <typename IN, typename OUT>
__global__ void __launch_bounds__(kThreads) topk_distill_any_kernel(const DistillParams p) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 red_max[kThreads / 32], red_sum[kThreads / 32], red_loss[kThreads / 32];
    uint32_t* ids = reinterpret_cast<uint32_t*>(smem);
    float* q = reinterpret_cast<float*>(ids + p.topk);
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const IN* zr = static_cast<const IN*>(p.logits) + row * p.ld;
    Words<kThreads, T0B_MAX_TOPK / kThreads> words;
    words.load(p, row, zr, true);
    float m = -INFINITY;
#pragma unroll 8
    for (uint32_t i = tid; i < p.cols; i += kThreads) m = fmaxf(m, to_float(zr[i]));
    block_max2<kThreads>(m, words.tmax, red_max);
    const Ref all(m, p.c);
    float s = 0.0f;
#pragma unroll 8
    for (uint32_t i = tid; i < p.cols; i += kThreads) s += exp2_approx(all.arg(to_float(zr[i]), p.c));
    const float tref = words.tmax == -INFINITY ? 0.0f : words.tmax;
    float tsum = words.sum(p, tref);
    block_sum2<kThreads>(s, tsum, red_sum);
    bool live = tsum > 0.0f || tsum != tsum;
    float2 cq = words.probs(p, tref, tsum, live, ids, q);
    if (m == -INFINITY && s == 0.0f) live = false;
    if (p.losses) {
        if (live) cq.x += words.cross(p, all);
        block_sum2<kThreads>(cq.x, cq.y, red_loss);
        if (tid == 0) p.losses[row] = live ? fmaf(cq.y, logf(s), cq.x) : 0.0f;
    }
    if (!p.dlogits) return;
    OUT* dr = static_cast<OUT*>(p.dlogits) + row * p.ld;
    const float a = live ? p.scale * (p.weights ? p.weights[row] : 1.0f) : 0.0f;
    const float inv = a / s;
#pragma unroll 4
    for (uint32_t i = tid; i < p.cols; i += kThreads) store_as(dr + i, live ? exp2_approx(all.arg(to_float(zr[i]), p.c)) * inv : 0.0f);
    if (!live) return;
    __syncthreads();
    words.gradient(p, all, a, s, 0, p.cols, ids, q, true, dr);
}

size_t words_bytes(const DistillParams& p) { return p.topk * 8ull + p.table * 4ull; }   // ids, q and the hash table

// One launch, behind the kernel in front of it in the stream (programmatic: its CTAs may be placed while that one drains).
template <typename K>
int32_t launch(t0b_ctx* ctx, K kernel, const DistillParams& p, uint32_t ctas, uint32_t threads, size_t smem, uint32_t cluster) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (ctx->pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return check_cuda(ctx, cudaLaunchKernelEx(&cfg, kernel, p), "cudaLaunchKernelEx(topk_distill)");
}

template <typename IN, typename OUT, int OWN>
int32_t launch_stream(t0b_ctx* ctx, const DistillParams& p, uint32_t rows) {
    auto kfn = topk_distill_stream_kernel<IN, OUT, OWN>;
    constexpr size_t kRing = static_cast<size_t>(kRingBatch) * kRingBatches * kStreamThreads * 16;
    static std::atomic<bool> configured[64];
    std::atomic<bool>& done = configured[ctx->device & 63];
    if (!done.load(std::memory_order_acquire)) {   // dynamic shared memory above 48 KB has to be asked for
        const int32_t rc = check_cuda(ctx, cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRing + T0B_MAX_TOPK * 8)), "cudaFuncSetAttribute(topk_distill)");
        if (rc != T0B_OK) return rc;
        done.store(true, std::memory_order_release);
    }
    return launch(ctx, kfn, p, rows, kStreamThreads, kRing + words_bytes(p), 1);
}

// Rows in registers, G groups a thread: the smallest G that holds the slice.
template <typename IN, typename OUT, int T, int OWN>
int32_t launch_registers(t0b_ctx* ctx, const DistillParams& p, uint32_t rows, uint32_t nranks) {
    const uint32_t g = (p.groups_per_cta + T - 1) / T, ctas = rows * nranks;
    const size_t smem = words_bytes(p);
    if (g <= 2) return launch(ctx, topk_distill_kernel<IN, OUT, 2, T, OWN>, p, ctas, T, smem, nranks);
    if (g <= 4) return launch(ctx, topk_distill_kernel<IN, OUT, 4, T, OWN>, p, ctas, T, smem, nranks);
    if constexpr (T == kThreads) {
        if (g > 8) return launch(ctx, topk_distill_kernel<IN, OUT, 16, T, OWN>, p, ctas, T, smem, nranks);
    }
    return launch(ctx, topk_distill_kernel<IN, OUT, 8, T, OWN>, p, ctas, T, smem, nranks);
}

template <typename IN, typename OUT>
int32_t run_distill(t0b_ctx* ctx, DistillParams p, uint32_t rows) {
    constexpr uint32_t N = Vec<IN>::kN;
    const uint32_t groups = p.cols / N + 1;
    const bool aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && reinterpret_cast<uintptr_t>(p.dlogits) % std::min<size_t>(16, N * sizeof(OUT)) == 0;
    if (!aligned) return launch(ctx, topk_distill_any_kernel<IN, OUT>, p, rows, kThreads, words_bytes(p), 1);
    // Rows that one CTA's registers hold stay there.  Longer ones are streamed when there is one for every SM (1001 x 32003
    // f32: 58 us against 69 us for clusters of two); with fewer rows clusters of CTAs share them: enough that a thread's
    // groups fit its registers, and more while SMs would idle and every thread still has two groups (24 x 32000 f32: 5.6 us).
    if (groups > kThreads * 16 && (rows >= static_cast<uint32_t>(ctx->num_sms) || groups > kMaxCluster * kThreads * 16)) {
        return p.topk <= kStreamThreads ? launch_stream<IN, OUT, 1>(ctx, p, rows) : launch_stream<IN, OUT, T0B_MAX_TOPK / kStreamThreads>(ctx, p, rows);
    }
    uint32_t nranks = 1;
    while (groups > nranks * kThreads * 16) nranks *= 2;
    while (nranks < kMaxCluster && static_cast<uint64_t>(rows) * nranks < static_cast<uint64_t>(ctx->num_sms) && groups >= nranks * kThreads * 4) nranks *= 2;
    if (static_cast<uint64_t>(rows) * nranks > 0x7fffffffull) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: %u rows are too many", rows);
    p.groups_per_cta = (groups + nranks - 1) / nranks;
    // The table takes 4000 x 9000 f32 with 100 words from 110 to 98 us; for up to four words the search costs no more (1127 x 1920
    // bf16, one word: 10.4 us either way), and streamed rows lose by it (4096 x 128000 bf16: 437 and 469 us).
    if (p.dlogits && p.topk > 4) {
        p.table = 32;
        p.table_shift = 27;
        while (p.table < 2 * p.topk) { p.table *= 2; --p.table_shift; }
    }
    // Short rows, many of them: CTAs of 128 threads, so that more rows are under way on an SM (8000 x 1000 f32: 24 us, 55 us
    // with 256 threads).
    if (nranks == 1 && groups <= 128 * 8 && p.topk <= 128 && rows >= 4u * static_cast<uint32_t>(ctx->num_sms)) return launch_registers<IN, OUT, 128, 1>(ctx, p, rows, 1);
    return p.topk <= kThreads ? launch_registers<IN, OUT, kThreads, 1>(ctx, p, rows, nranks)
                              : launch_registers<IN, OUT, kThreads, T0B_MAX_TOPK / kThreads>(ctx, p, rows, nranks);
}

}  // namespace

extern "C" {

int32_t t0b_topk_distill(t0b_ctx* ctx, uint64_t logits, int32_t logits_dtype, uint64_t ids, uint64_t teacher, uint64_t row_weights,
                         uint64_t losses, uint64_t dlogits, int32_t grad_dtype, uint32_t rows, uint32_t cols, uint64_t ld,
                         uint32_t topk, uint64_t ldk, float temperature, float scale, int32_t async) try {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (rows == 0) return T0B_OK;
    if (logits_dtype != T0B_OUT_F32 && logits_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: unknown logits_dtype %d", logits_dtype);
    if (dlogits && grad_dtype != T0B_OUT_F32 && grad_dtype != T0B_OUT_BF16) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: unknown grad_dtype %d", grad_dtype);
    if (!logits || !ids || !teacher || (!losses && !dlogits)) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: null pointer");
    if (cols == 0 || cols > 0x7fffff00u || ld < cols) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: %u columns with a pitch of %llu", cols, static_cast<unsigned long long>(ld));
    if (topk == 0 || topk > T0B_MAX_TOPK || ldk < topk)
        return set_error(ctx, T0B_ERR_INVALID, "topk_distill: topk %u is outside 1..%d, or its pitch %llu is smaller", topk, T0B_MAX_TOPK, static_cast<unsigned long long>(ldk));
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(1.4426950408889634f / temperature) || !std::isfinite(scale))
        return set_error(ctx, T0B_ERR_INVALID, "topk_distill: temperature %g and its inverse must be positive and finite, scale %g finite", temperature, scale);
    if (!std::isfinite(scale / temperature)) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: scale %g over temperature %g is not finite", scale, temperature);
    const size_t ie = logits_dtype == T0B_OUT_BF16 ? 2 : 4, oe = grad_dtype == T0B_OUT_BF16 ? 2 : 4;
    if (logits % ie || (dlogits && dlogits % oe) || ids % 4 || teacher % 4 || losses % 4 || row_weights % 4)
        return set_error(ctx, T0B_ERR_INVALID, "topk_distill: a pointer is not aligned to its element");
    if (dlogits == logits && ie != oe) return set_error(ctx, T0B_ERR_INVALID, "topk_distill: a gradient in the place of the logits needs their type");
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    rc = check_fits(ctx, "topk_distill", {{"logits", logits, span_bytes(rows, ld, cols, ie)}, {"dlogits", dlogits, span_bytes(rows, ld, cols, oe)},
                                          {"ids", ids, span_bytes(rows, ldk, topk, 4)}, {"teacher", teacher, span_bytes(rows, ldk, topk, 4)},
                                          {"losses", losses, rows * 4ull}, {"row_weights", row_weights, rows * 4ull}});
    if (rc != T0B_OK) return rc;

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
    p.status = ctx->status_dev;
    if (ie == 2) rc = oe == 2 ? run_distill<__nv_bfloat16, __nv_bfloat16>(ctx, p, rows) : run_distill<__nv_bfloat16, float>(ctx, p, rows);
    else rc = oe == 2 ? run_distill<float, __nv_bfloat16>(ctx, p, rows) : run_distill<float, float>(ctx, p, rows);
    if (rc != T0B_OK) return rc;
    return finish(ctx, async, "topk_distill");
} catch (...) {
    return T0B_ERR_NOMEM;   // no C++ exception leaves a C entry
}

}  // extern "C"
