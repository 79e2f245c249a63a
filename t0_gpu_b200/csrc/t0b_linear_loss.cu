// The vocabulary losses straight from the hidden states and the head, without the [rows, vocab] logits:
//   z = x * head,  p = softmax(z / T),  loss_r = sum_k q_rk (log q_rk - log p_r,id_rk)
// with a sparse target distribution q per row: one word with q = 1 (cross entropy), or the softmax of a teacher's top logits.
//   dz = (p sum(q) - q) * scale * weight_r / T,   dx = dz * head^T,   dhead = x^T * dz
// The vocabulary goes through the tensor cores in tiles whose epilogue keeps the maximum and the sum of exponentials of every
// row's part (head_gemm); a join over the parts gives the row's log-sum-exp and its loss.  That is all that an evaluation
// does: 2 rows dim vocab operations, and nothing of the size rows x vocab is written.
// For the gradient the same epilogue also leaves the exponentials of a piece of the rows, relative to their part's maximum,
// in 16 bits (at most 1 GiB, or what 256 rows take, whatever the number of rows); one pass turns them into dz in place, and two products give dx
// and the head's gradient, which sums over the pieces in f32.  6 rows dim vocab operations in all: computing the exponentials
// anew once the sums are known would cost 8, and the pass over 16-bit exponentials costs 4 bytes per element against
// 2 dim operations (at dim 4096: 4 % of the step instead of 33 %).
// Roundings: products of bf16 operands with f32 sums; exponentials to fp16 (HeadParams), dz to bf16 -- the operand type of
// the two gradient products -- computed in f32 from the f32 logit at every word of q, where it is largest.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "ptx_sm100.cuh"
#include "t0b_internal.hpp"

using namespace t0b;

namespace {

constexpr uint32_t kNoWord = 0xffffffffu;
constexpr uint64_t kPieceBytes = 1ull << 30;       // exponentials of one piece of rows
constexpr uint64_t kPartBytes = 1ull << 28;        // per-part statistics of one piece of rows

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2, float c) {
    const float mm = fmaxf(m, m2);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    s = s * exp2_approx((m - ref) * c) + s2 * exp2_approx((m2 - ref) * c);
    m = mm;
}

// --------------------------------------------------------------------------------------------------- rows as operands
__device__ __forceinline__ uint4 pack_bf16x8(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Columns c ... c + 7 of a row of `cols` elements as bf16, zeros behind its end.
template <typename IN>
__device__ __forceinline__ uint4 operand_group(const IN* row, uint32_t c, uint32_t cols, bool vec) {
    const IN* src = row + c;
    if constexpr (sizeof(IN) == 2) {
        if (vec && c + 8 <= cols) return *reinterpret_cast<const uint4*>(src);
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t a = c + 2 * e < cols ? *reinterpret_cast<const uint16_t*>(src + 2 * e) : 0u;
            const uint32_t b = c + 2 * e + 1 < cols ? *reinterpret_cast<const uint16_t*>(src + 2 * e + 1) : 0u;
            w[e] = a | (b << 16);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        float v[8];
        if (vec && c + 8 <= cols) {
            const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? static_cast<float>(src[e]) : 0.0f;
        }
        return pack_bf16x8(v);
    }
}
template <typename IN>
__device__ __forceinline__ bool rows_vec(const IN* in, unsigned long long ld) {
    return (reinterpret_cast<uintptr_t>(in) & 15) == 0 && ld % (16 / sizeof(IN)) == 0;
}

// out[r, c] = bf16(in[r, c]), rows of `cols` elements at a pitch of whole 16 bytes; a row without a target is written as zeros,
// whatever it holds (its hidden state may be anything, and 0 * NaN would reach the head's gradient).
template <typename IN>
__global__ void __launch_bounds__(256) pack_rows_kernel(const IN* in, unsigned long long ld, __nv_bfloat16* out, uint32_t ld_out, uint32_t rows,
                                                        uint32_t cols, const uint32_t* targets, uint32_t vocab) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint32_t per_row = ld_out / 8;
    const unsigned long long total = static_cast<unsigned long long>(rows) * per_row;
    const bool vec = rows_vec(in, ld);
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t r = static_cast<uint32_t>(i / per_row), c = static_cast<uint32_t>(i % per_row) * 8;
        const uint4 o = targets[r] < vocab ? operand_group(in + r * ld, c, cols, vec) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(out + static_cast<unsigned long long>(r) * ld_out + c) = o;
    }
}

// The same copy of a bf16 matrix whose rows start off 16-byte boundaries (a head with an odd vocabulary, [dim, vocab]): a warp
// reads whole 16-byte chunks of the source, a lane shifts its chunk and its neighbour's into the 16 bytes it writes.  Chunks
// that reach over the matrix' ends are read by element.  2048 x 50257: 206 MB each way, bound by HBM.
// HIGH rows to a block: 8 for narrow matrices (37980 x 157: 9 us, 41 us with 1), else 1 (1664 x 32028: 43 us, and 50 us with
// the row per thread).
template <uint32_t HIGH>
__global__ void __launch_bounds__(256) pack_shifted_kernel(const __nv_bfloat16* in, unsigned long long ld, __nv_bfloat16* out, uint32_t ld_out,
                                                           uint32_t rows, uint32_t cols) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t c = (blockIdx.x * (256 / HIGH) + threadIdx.x) * 8;   // a warp's columns are neighbours
    const uint64_t begin = reinterpret_cast<uint64_t>(in), end = begin + ((rows - 1ull) * ld + cols) * 2;
    auto load = [&](uint64_t addr) {
        return addr >= begin && addr + 16 <= end ? __ldcs(reinterpret_cast<const uint4*>(addr)) : make_uint4(0, 0, 0, 0);
    };
    for (uint32_t r = HIGH == 1 ? blockIdx.y : blockIdx.y * HIGH + threadIdx.y; r < rows; r += gridDim.y * HIGH) {
        const uint64_t at = begin + (r * ld + c) * 2, chunk = at & ~15ull;
        const uint32_t shift = static_cast<uint32_t>(at & 15);
        const uint4 a = load(chunk);
        uint4 b;
        b.x = __shfl_down_sync(0xffffffffu, a.x, 1);
        b.y = __shfl_down_sync(0xffffffffu, a.y, 1);
        b.z = __shfl_down_sync(0xffffffffu, a.z, 1);
        b.w = __shfl_down_sync(0xffffffffu, a.w, 1);
        if (c >= ld_out) continue;
        if (lane == 31) b = load(chunk + 16);
        uint4 o;
        if (chunk < begin || chunk + (shift ? 32 : 16) > end || c + 8 > cols) {
            o = operand_group(in + r * ld, c, cols, false);
        } else {
            uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 6; ++e) w[e] = (shift & 8) ? w[e + 2] : w[e];
#pragma unroll
            for (int e = 0; e < 5; ++e) w[e] = (shift & 4) ? w[e + 1] : w[e];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __funnelshift_r(w[e], w[e + 1], (shift & 2) * 8);
            o = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(out + static_cast<unsigned long long>(r) * ld_out + c) = o;
    }
}

// ------------------------------------------------------------------------------------------------ the teacher's words
// One row per threadIdx.y, one word per threadIdx.x (P = a power of two >= topk): q = softmax(t / T) over the words that are
// there, entropy = sum q log q, and the words in ascending order of id (what the head's epilogue searches).  A word named
// more than once keeps its first place with the sum of its q; the other places get q = -1.  Then the row's hidden state is
// copied as pack_rows_kernel does it (x_out null: no copy is needed).
template <typename IN>
__global__ void __launch_bounds__(1024) teacher_words_kernel(const uint32_t* ids, const float* teacher, unsigned long long ldk, uint32_t rows,
                                                             uint32_t topk, uint32_t vocab, float inv_t, uint32_t* out_ids, float* out_q,
                                                             float* entropy, uint32_t* live, int* status, const IN* x, unsigned long long ldx,
                                                             __nv_bfloat16* x_out, uint32_t ldx_out, uint32_t dim) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t P = blockDim.x, k = threadIdx.x, y = threadIdx.y;
    unsigned long long* key = reinterpret_cast<unsigned long long*>(smem) + static_cast<size_t>(y) * P;
    float* val = reinterpret_cast<float*>(smem + static_cast<size_t>(blockDim.y) * P * 8) + static_cast<size_t>(y) * P;
    const uint32_t row = blockIdx.x * blockDim.y + y;
    const bool in = row < rows && k < topk;
    uint32_t id = kNoWord;
    float t = -INFINITY;
    if (in) {
        id = ids[row * ldk + k];
        t = teacher[row * ldk + k];
        if (id != kNoWord && id >= vocab) {
            *reinterpret_cast<volatile int*>(status) = kDevBadIndex;   // the word is left out
            id = kNoWord;
        }
        if (id == kNoWord) t = -INFINITY;
    }
    // Over the row: within its warps by shuffles (P >= 32), then over the warps.
    auto reduce = [&](float v, bool is_max) -> float {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float u = __shfl_xor_sync(0xffffffffu, v, o);
            v = is_max ? fmaxf(v, u) : v + u;
        }
        if (P == 32) return v;
        __syncthreads();
        if ((k & 31) == 0) val[k >> 5] = v;
        __syncthreads();
        v = val[0];
        for (uint32_t i = 1; i < P / 32; ++i) v = is_max ? fmaxf(v, val[i]) : v + val[i];
        return v;
    };
    const float mx = reduce(t, true);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    const float e = id == kNoWord ? 0.0f : expf((t - ref) * inv_t);
    const float sum = reduce(e, false);
    const bool some = sum > 0.0f || sum != sum;
    const float lq = (t - ref) * inv_t - logf(sum);
    const float q = (some && id != kNoWord) ? e / sum : 0.0f;
    const float ent = reduce(q != 0.0f ? q * lq : 0.0f, false);
    __syncthreads();
    key[k] = (static_cast<unsigned long long>(some ? id : kNoWord) << 32) | k;
    val[k] = q;
    __syncthreads();
    for (uint32_t size = 2; size <= P; size <<= 1)
        for (uint32_t stride = size >> 1; stride > 0; stride >>= 1) {
            const uint32_t other = k ^ stride;
            if (other > k) {
                const unsigned long long a = key[k], b = key[other];
                if ((a > b) == ((k & size) == 0)) {
                    key[k] = b;
                    key[other] = a;
                }
            }
            if (stride >= 32) __syncthreads();   // partners in one warp: the warp's own order is enough
            else __syncwarp();
            if (stride == 1) __syncthreads();
        }
    if (in) {
        const uint32_t my = static_cast<uint32_t>(key[k] >> 32);
        float qs = val[static_cast<uint32_t>(key[k])];
        if (my != kNoWord) {
            if (k > 0 && static_cast<uint32_t>(key[k - 1] >> 32) == my) qs = -1.0f;
            else
                for (uint32_t i = k + 1; i < P && static_cast<uint32_t>(key[i] >> 32) == my; ++i) qs += val[static_cast<uint32_t>(key[i])];
        }
        out_ids[static_cast<size_t>(row) * topk + k] = my;
        out_q[static_cast<size_t>(row) * topk + k] = qs;
        if (k == 0) {
            entropy[row] = some ? ent : 0.0f;
            live[row] = some ? 1u : 0u;
        }
    }
    if (x_out && row < rows) {
        const bool vec = rows_vec(x, ldx);
        for (uint32_t c = k * 8; c < ldx_out; c += P * 8)
            *reinterpret_cast<uint4*>(x_out + static_cast<unsigned long long>(row) * ldx_out + c) =
                some ? operand_group(x + row * ldx, c, dim, vec) : make_uint4(0, 0, 0, 0);
    }
}

// out[r, c] = bf16(acc[r, c]): the head's gradient summed in f32 over several pieces, rounded once.
__global__ void __launch_bounds__(256) round_rows_kernel(const float* acc, uint32_t ld_acc, __nv_bfloat16* out,
                                                         unsigned long long ld, uint32_t rows, uint32_t cols) {
    ptx::grid_dependency_wait();
    const uint32_t per_row = (cols + 7) / 8;
    const unsigned long long total = static_cast<unsigned long long>(rows) * per_row;
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ld % 8 == 0;
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t r = static_cast<uint32_t>(i / per_row), c = static_cast<uint32_t>(i % per_row) * 8;
        const float4* src = reinterpret_cast<const float4*>(acc + static_cast<unsigned long long>(r) * ld_acc + c);   // pitch: whole 8 elements
        const float4 a = __ldcs(src), b = __ldcs(src + 1);
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        __nv_bfloat16* dst = out + r * ld + c;
        if (vec && c + 8 <= cols) {
            *reinterpret_cast<uint4*>(dst) = pack_bf16x8(v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < cols) dst[e] = __float2bfloat16_rn(v[e]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ rows with a target
// Which rows have a target, in order: row_of[i] = the i-th of them, place_of[r] = its place or kNoWord, count = how many.  The
// products then run over those rows alone, and count stays on the device.  One block: thread t looks at the rows
// [t * per, (t + 1) * per).  Rows that are left out get their losses here.
__global__ void __launch_bounds__(1024) live_rows_kernel(const uint32_t* targets, const uint32_t* live, uint32_t vocab, uint32_t rows, uint32_t* row_of,
                                                         uint32_t* place_of, int* count, float* losses, float* lse, int* status) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    __shared__ uint32_t warp_sums[32];
    const uint32_t per = (rows + 1023) / 1024, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t lo = min(rows, threadIdx.x * per), hi = min(rows, lo + per);
    uint32_t mine = 0;
    for (uint32_t r = lo; r < hi; ++r) mine += live ? (live[r] != 0) : (targets[r] < vocab);
    uint32_t upto = mine;   // inclusive sum over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < 32; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    uint32_t at = before + upto - mine;
    for (uint32_t r = lo; r < hi; ++r) {
        const bool on = live ? (live[r] != 0) : (targets[r] < vocab);
        if (on) row_of[at] = r;
        else {
            if (losses) losses[r] = 0.0f;
            if (lse) lse[r] = 0.0f;
            if (!live && targets[r] != kNoWord) *reinterpret_cast<volatile int*>(status) = kDevBadIndex;
        }
        place_of[r] = on ? at++ : kNoWord;
    }
    if (threadIdx.x == 0) *count = static_cast<int>(all);
}

// The rows with a target, gathered as bf16 operand rows, and 64 rows of zeros behind the last: the head's gradient contracts
// whole 64-row blocks, counted from the start of a piece.
template <typename IN>
__global__ void __launch_bounds__(256) gather_rows_kernel(const IN* in, unsigned long long ld, __nv_bfloat16* out, uint32_t ld_out, uint32_t rows,
                                                          uint32_t cols, const uint32_t* row_of, const int* count) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint32_t per_row = ld_out / 8, n = static_cast<uint32_t>(*count), padded = min(rows, n + 64);
    const unsigned long long total = static_cast<unsigned long long>(padded) * per_row;
    const bool vec = rows_vec(in, ld);
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t r = static_cast<uint32_t>(i / per_row), c = static_cast<uint32_t>(i % per_row) * 8;
        const uint4 o = r < n ? operand_group(in + row_of[r] * ld, c, cols, vec) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(out + static_cast<unsigned long long>(r) * ld_out + c) = o;
    }
}

// dx[r, :] = the gathered gradient at the row's place, or zeros.  T: the gradient's type, moved as it is.
template <typename T>
__global__ void __launch_bounds__(256) spread_rows_kernel(const T* in, uint32_t ld_in, T* out, unsigned long long ld, uint32_t rows, uint32_t cols,
                                                          const uint32_t* place_of) {
    ptx::grid_dependency_wait();
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t per_row = (cols + N - 1) / N;
    const unsigned long long total = static_cast<unsigned long long>(rows) * per_row;
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ld % N == 0;
    for (unsigned long long i = blockIdx.x * 256ull + threadIdx.x; i < total; i += gridDim.x * 256ull) {
        const uint32_t r = static_cast<uint32_t>(i / per_row), c = static_cast<uint32_t>(i % per_row) * N;
        const uint32_t at = place_of[r];
        uint4 v = make_uint4(0, 0, 0, 0);
        if (at != kNoWord) v = *reinterpret_cast<const uint4*>(in + static_cast<unsigned long long>(at) * ld_in + c);   // pitch: whole 16 bytes
        T* dst = out + r * ld + c;
        if (vec && c + N <= cols) {
            *reinterpret_cast<uint4*>(dst) = v;
        } else {
            const T* e = reinterpret_cast<const T*>(&v);
            for (uint32_t j = 0; j < N && c + j < cols; ++j) dst[j] = e[j];
        }
    }
}

// ------------------------------------------------------------------------------------------------- joining the parts
// What the join and the gradient pass know about the targets of a row.
struct Targets {
    const uint32_t* ids;      // [rows][n_ids], by row of the call like q, entropy and live
    const float* q;           // [rows][n_ids], null: cross entropy (one word, q = 1)
    const float* entropy;     // [rows], with q
    const uint32_t* live;     // [rows], with q
    const float* z_sel;       // [rows of the piece][n_ids]
    uint32_t n_ids, vocab;
    // Products over the rows with a target alone: row i of a piece is row row_of[row0 + i] of the call, and the piece has
    // count - row0 of them.  Null: row i is row row0 + i.
    const uint32_t* row_of;
    const int* count;
    uint32_t row0;
    __device__ __forceinline__ uint32_t rows_here(uint32_t most) const {
        return row_of ? static_cast<uint32_t>(max(0, min(static_cast<int>(most), *count - static_cast<int>(row0)))) : most;
    }
    __device__ __forceinline__ uint32_t row(uint32_t i) const { return row_of ? row_of[row0 + i] : row0 + i; }
};
__device__ __forceinline__ bool row_live(const Targets& t, uint32_t row) { return t.q ? t.live[row] != 0 : t.ids[row] < t.vocab; }

// One warp: the loss and log-sum-exp of row i of the piece, row r of the call, from its (max z, sum of exp).
__device__ __forceinline__ void finish_row(float m, float s, uint32_t i, uint32_t r, float inv_t, const Targets& tg, float* losses, float* lse_out,
                                           int* status) {
    const uint32_t lane = threadIdx.x & 31;
    const bool none = m == -INFINITY && s == 0.0f;       // every logit is -inf: the row has no distribution
    const bool live = row_live(tg, r) && !none;
    const float log_s = logf(s);
    float cross = 0.0f;
    if (live) {
        const float* z = tg.z_sel + static_cast<size_t>(i) * tg.n_ids;
        if (tg.q) {
            for (uint32_t k = lane; k < tg.n_ids; k += 32) {
                const float q = tg.q[static_cast<size_t>(r) * tg.n_ids + k];
                if (tg.ids[static_cast<size_t>(r) * tg.n_ids + k] == kNoWord || q == 0.0f || q < 0.0f) continue;
                cross += q * (log_s - (z[k] - m) * inv_t);
            }
            cross = warp_sum(cross) + tg.entropy[r];
        } else {
            cross = log_s - (z[0] - m) * inv_t;
        }
    }
    if (lane == 0) {
        if (losses) losses[r] = live ? cross : 0.0f;
        if (lse_out) lse_out[r] = live ? m * inv_t + log_s : 0.0f;
        if (!tg.q && tg.ids[r] >= tg.vocab && tg.ids[r] != kNoWord) *reinterpret_cast<volatile int*>(status) = kDevBadIndex;
    }
}

// One block per 32 rows: warps walk the parts (a warp's load is 32 neighbouring rows of one part), the warps' results meet in
// shared memory, then warp i finishes row i: stats[row] = (max z, sum of exp), the loss and log-sum-exp.
__global__ void __launch_bounds__(1024) join_parts_kernel(const float2* part, unsigned long long part_ld, uint32_t parts, uint32_t rows,
                                                          float c, float inv_t, Targets tg, float2* stats,
                                                          float* losses, float* lse_out, int* status) {
    __shared__ float2 sh[32][33];
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    rows = tg.rows_here(rows);
    if (blockIdx.x * 32 >= rows) return;
    const uint32_t at = blockIdx.x * 32 + lane;
    float m = -INFINITY, s = 0.0f;
    if (at < rows) {
        for (uint32_t i = warp; i < parts; i += 128) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = i + 32 * u < parts ? part[(i + 32 * u) * part_ld + at] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; ++u) join_stats(m, s, v[u].x, v[u].y, c);
        }
    }
    sh[warp][lane] = make_float2(m, s);
    __syncthreads();
    const uint32_t i = blockIdx.x * 32 + warp;   // the row of the piece, and r of the call
    if (i >= rows) return;
    const uint32_t r = tg.row(i);
    m = sh[lane][warp].x;
    s = sh[lane][warp].y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        join_stats(m, s, m2, s2, c);
    }
    finish_row(m, s, i, r, inv_t, tg, losses, lse_out, status);
    if (lane == 0) stats[i] = make_float2(m, s);
}

// ---------------------------------------------------------------------------------------------------- the gradient of z
// u (fp16, kHeadUScale relative to its part's maximum) becomes dz (bf16) in place: a block takes kGradCols columns of one row.  The
// words of the targets are written last, from their f32 logit.  Bound by HBM: 2 bytes in, 2 bytes out per element (4096 x
// 128000: 358 us, 5.9 TB/s).  Two small steps ride along where their own launch would cost more than they do:
//   JOIN   every block joins its row's parts itself, and the row's first block finishes the loss (join_parts_kernel is not
//          launched): for few rows or few parts
//   cp.x   the row's first block copies the hidden state, or zeros in a row that is left out, for the head's gradient
// Where that copy was made before the logits were known, the row's first block clears it in a row whose logits are all -inf:
// an infinity in the hidden state would meet dz = 0 in the head's gradient.
constexpr int kGradVecs = 4;
constexpr uint32_t kGradCols = 256 * 8 * kGradVecs;
struct JoinParams { uint32_t parts; float inv_t; float *losses, *lse; int* status; };
struct CopyParams { const __nv_bfloat16* x; unsigned long long ldx; __nv_bfloat16* out; uint32_t ld_out, dim; };   // out null: no gradient of the head
template <bool JOIN>
__global__ void __launch_bounds__(256) dz_kernel(__half* u, unsigned long long ldu, uint32_t rows, uint32_t y0, const float2* part,
                                                 unsigned long long part_ld, uint32_t part_shift, const float2* stats,
                                                 const float* weights, float scale, float c, Targets tg, JoinParams jp, CopyParams cp) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint32_t i = y0 + blockIdx.y;          // the row of the piece, and r of the call
    const uint32_t c0 = blockIdx.x * kGradCols;
    const uint32_t n = tg.rows_here(rows);
    const bool behind = i >= n;                  // zeros up to a whole 64-row block: the head's gradient reads it
    if (behind && i >= max(64u, (n + 63) / 64 * 64)) return;
    const uint32_t r = behind ? 0 : tg.row(i);
    __half* ur = u + i * ldu;
    __nv_bfloat16* gr = reinterpret_cast<__nv_bfloat16*>(ur);
    const bool wanted = !behind && row_live(tg, r);
    uint4 raw[kGradVecs];
    float top[kGradVecs];
#pragma unroll
    for (int v = 0; v < kGradVecs; ++v) {
        const uint32_t col = c0 + (v * 256 + threadIdx.x) * 8;
        if (wanted && col < ldu) {
            raw[v] = __ldcs(reinterpret_cast<const uint4*>(ur + col));
            top[v] = part[(col >> part_shift) * part_ld + i].x;
        }
    }
    // The first 2048 columns of the hidden state are asked for with the exponentials; whether they are copied is known later.
    const bool first = cp.out && blockIdx.x == 0 && !behind;
    const bool copy_x = first && cp.x != nullptr, vec_x = copy_x && rows_vec(cp.x, cp.ldx);
    uint4 x0 = make_uint4(0, 0, 0, 0);
    if (copy_x && wanted && threadIdx.x * 8 < cp.ld_out) x0 = operand_group(cp.x + r * cp.ldx, threadIdx.x * 8, cp.dim, vec_x);
    float2 st = make_float2(0.0f, 1.0f);
    if constexpr (JOIN) {
        __shared__ float2 sh[8];
        float m = -INFINITY, s = 0.0f;
        if (!behind)
            for (uint32_t k = threadIdx.x; k < jp.parts; k += 256) {
                const float2 v = part[k * part_ld + i];
                join_stats(m, s, v.x, v.y, c);
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
            join_stats(m, s, m2, s2, c);
        }
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(m, s);
        __syncthreads();
        m = sh[0].x;
        s = sh[0].y;
        for (int w = 1; w < 8; ++w) join_stats(m, s, sh[w].x, sh[w].y, c);
        if (!behind) {
            st = make_float2(m, s);
            if (blockIdx.x == 0 && threadIdx.x < 32) finish_row(m, s, i, r, jp.inv_t, tg, jp.losses, jp.lse, jp.status);
        }
    } else {
        if (!behind) st = stats[i];
    }
    const bool live = wanted && !(st.x == -INFINITY && st.y == 0.0f);
    const float a = live ? scale * (weights ? weights[r] : 1.0f) : 0.0f;
    const float inv = 1.0f / st.y;
    if (copy_x || (first && wanted && !live)) {
        __nv_bfloat16* xr = cp.out + static_cast<unsigned long long>(tg.row0 + i) * cp.ld_out;
        for (uint32_t col = threadIdx.x * 8; col < cp.ld_out; col += 256 * 8) {
            uint4 o = make_uint4(0, 0, 0, 0);
            if (copy_x && live) o = col < 256 * 8 ? x0 : operand_group(cp.x + r * cp.ldx, col, cp.dim, vec_x);
            *reinterpret_cast<uint4*>(xr + col) = o;
        }
    }
#pragma unroll
    for (int v = 0; v < kGradVecs; ++v) {
        const uint32_t col = c0 + (v * 256 + threadIdx.x) * 8;
        if (col >= ldu) continue;
        uint4 o = make_uint4(0, 0, 0, 0);
        if (live) {
            const float f = a * (exp2_approx((top[v] - st.x) * c) * inv) * (1.0f / kHeadUScale);
            const uint32_t w[4] = {raw[v].x, raw[v].y, raw[v].z, raw[v].w};
            float g[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                g[2 * e] = t.x * f;
                g[2 * e + 1] = t.y * f;
            }
            o = pack_bf16x8(g);
        }
        *reinterpret_cast<uint4*>(gr + col) = o;
    }
    if (!live) return;
    __syncthreads();
    const float* z = tg.z_sel + static_cast<size_t>(i) * tg.n_ids;
    for (uint32_t k = threadIdx.x; k < tg.n_ids; k += 256) {
        const size_t at = static_cast<size_t>(r) * tg.n_ids + k;
        const uint32_t id = tg.ids[at];
        if (id - c0 >= kGradCols || id >= tg.vocab) continue;
        const float q = tg.q ? tg.q[at] : 1.0f;
        if (q < 0.0f) continue;
        gr[id] = __float2bfloat16_rn(a * (exp2_approx((z[k] - st.x) * c) * inv - q));
    }
}

// Programmatic launch: a kernel's blocks may be placed while the one before drains; every kernel here waits for it before it
// touches memory.
template <typename... P, typename... A>
void launch(t0b_ctx* ctx, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);   // an error stays with the runtime until finish() asks
}

uint64_t align256(uint64_t x) { return (x + 255) & ~255ull; }
uint64_t round8(uint64_t x) { return (x + 7) & ~7ull; }

// Everything a call will do, from its arguments alone: pieces, tile, operand copies, scratch layout.
struct Plan {
    bool grads, dx, dw;
    uint32_t piece, pieces;
    HeadPlan head;
    uint32_t parts;
    uint64_t part_ld;
    uint64_t ldu;
    bool copy_x, copy_w;               // before the head's product
    bool late_x;                       // the copy of x for the head's gradient (which always reads one) is made by dz_kernel; the head reads x itself
    bool join_in_dz;
    bool gather;                       // the products run over the rows with a target alone
    uint64_t ld_dxg;
    uint64_t row_of, place_of, count, dxg;
    uint64_t ldx, ldw;                 // pitches of the operands as the products read them
    uint64_t w_rows, w_cols;
    bool acc_dw;                       // bf16 gradient of the head over several pieces: summed in f32 in the scratch
    uint64_t ld_acc;
    uint64_t x, w, ids, q, entropy, live, z_sel, part, stats, u, acc, slabs;   // offsets
    uint64_t slab_bytes, total;
};

bool tma_ok(uint64_t ptr, uint64_t ld) { return ptr % 16 == 0 && ld % 8 == 0; }

InnerGemm dx_gemm(const t0b_linear_loss& d, const Plan& p, uint64_t u, uint64_t w, uint64_t base, uint32_t r0, uint32_t n) {
    InnerGemm g{};
    const uint64_t out = p.gather ? base + p.dxg : d.dx, ld = p.gather ? p.ld_dxg : d.lddx;
    if (p.gather) { g.dyn_rows = base + p.count; g.dyn_off = static_cast<int>(r0); }
    g.trans_a = 0;
    g.trans_b = d.trans_w ? 0 : 1;
    g.a = u; g.b = w;
    g.c = out + static_cast<uint64_t>(r0) * ld * (d.dx_dtype == T0B_OUT_BF16 ? 2 : 4);
    g.m = n; g.n = d.dim; g.k = d.vocab;
    g.lda = p.ldu; g.ldb = p.ldw; g.ldc = ld;
    g.out_bf16 = d.dx_dtype == T0B_OUT_BF16;
    return g;
}

InnerGemm dw_gemm(const t0b_linear_loss& d, const Plan& p, uint64_t u, uint64_t x, uint64_t base, uint32_t r0, uint32_t n) {
    InnerGemm g{};
    const uint64_t acc = base + p.acc;
    if (p.gather) { g.dyn_rows = base + p.count; g.dyn_off = static_cast<int>(r0); g.dyn_k = 1; }
    const uint64_t xr = x + static_cast<uint64_t>(r0) * p.ldx * 2;
    g.trans_a = 1;
    g.trans_b = 0;
    if (d.trans_w) { g.a = u; g.b = xr; g.m = d.vocab; g.n = d.dim; g.lda = p.ldu; g.ldb = p.ldx; }
    else { g.a = xr; g.b = u; g.m = d.dim; g.n = d.vocab; g.lda = p.ldx; g.ldb = p.ldu; }
    g.k = n;
    g.c = p.acc_dw ? acc : d.dw;
    g.ldc = p.acc_dw ? p.ld_acc : d.lddw;
    g.out_bf16 = !p.acc_dw && d.dw_dtype == T0B_OUT_BF16;
    g.accumulate = r0 > 0;
    g.head_grad = true;
    return g;
}

Plan make_plan(t0b_ctx* ctx, const t0b_linear_loss& d, uint32_t n_ids, bool teacher) {
    Plan p{};
    p.dx = d.dx != 0;
    p.dw = d.dw != 0;
    p.grads = p.dx || p.dw;
    p.ldu = round8(d.vocab);
    // Pieces of rows: whole 256-row tiles, as even as they come.
    uint64_t fit = p.grads ? kPieceBytes / (p.ldu * 2) : kPartBytes / ((d.vocab / 64 + 1) * 8ull);
    fit = std::max<uint64_t>(256, fit / 256 * 256);
    if (d.piece_rows > 0) fit = d.piece_rows;
    p.pieces = static_cast<uint32_t>((d.rows + fit - 1) / fit);
    p.piece = (d.rows + p.pieces - 1) / p.pieces;
    if (p.pieces > 1 && d.piece_rows == 0) p.piece = (p.piece + 255) / 256 * 256;
    if (p.pieces > 1 && d.piece_rows > 0) p.piece = d.piece_rows;
    p.pieces = (d.rows + p.piece - 1) / p.piece;
    p.head = head_plan(ctx, p.piece, d.vocab, d.dim);
    p.parts = (d.vocab + p.head.part_cols - 1) / p.head.part_cols;
    p.part_ld = (p.piece + 31ull) / 32 * 32;
    // Up to a tile of rows costs the same with and without the rows that are left out; the losses alone of a small product
    // cost less than finding the rows (two kernels, 5 us).
    p.gather = d.rows > 256 && (p.grads || 2.0 * d.rows * d.dim * d.vocab >= 5e10);
    p.copy_x = p.gather || d.x_dtype != T0B_OUT_BF16 || !tma_ok(d.x, d.ldx);
    p.late_x = p.dw && !p.copy_x;
    p.ldx = p.copy_x || p.late_x ? round8(d.dim) : d.ldx;
    p.w_rows = d.trans_w ? d.vocab : d.dim;
    p.w_cols = d.trans_w ? d.dim : d.vocab;
    // A part's (maximum, sum) is 8 bytes of a 32-byte sector to a block that joins one row: up to 16 MB of them in all.
    p.join_in_dz = p.grads && p.piece * ((p.ldu + kGradCols - 1) / kGradCols) * p.parts * 32ull <= (16ull << 20);
    p.copy_w = !tma_ok(d.w, d.ldw);
    p.ldw = p.copy_w ? round8(p.w_cols) : d.ldw;
    p.acc_dw = p.dw && p.pieces > 1 && d.dw_dtype == T0B_OUT_BF16;
    p.ld_acc = round8(p.w_cols);
    uint64_t off = 0;
    auto take = [&](uint64_t bytes) { const uint64_t at = off; off += align256(bytes); return at; };
    const uint64_t rows = d.rows;
    p.stats = take(rows * 8);
    p.z_sel = take(rows * n_ids * 4);
    if (teacher) {
        p.ids = take(rows * n_ids * 4);
        p.q = take(rows * n_ids * 4);
        p.entropy = take(rows * 4);
        p.live = take(rows * 4);
    }
    if (p.copy_x || p.late_x) p.x = take(rows * p.ldx * 2);
    if (p.copy_w) p.w = take(p.w_rows * p.ldw * 2);
    if (p.gather) {
        p.row_of = take(rows * 4);
        p.place_of = take(rows * 4);
        p.count = take(4);
        p.ld_dxg = round8(d.dim);
        if (p.dx) p.dxg = take(rows * p.ld_dxg * (d.dx_dtype == T0B_OUT_BF16 ? 2 : 4));
    }
    p.part = take(p.parts * p.part_ld * 8);
    if (p.grads) p.u = take(p.piece * p.ldu * 2);
    if (p.acc_dw) p.acc = take(p.w_rows * p.ld_acc * 4);
    // Slabs of a split contraction, for whichever product of whichever piece wants most; the products run one after another.
    for (uint32_t r0 = 0; p.grads && r0 < d.rows; r0 += p.piece) {
        const uint32_t n = std::min(p.piece, d.rows - r0);
        if (r0 > 0 && n == p.piece) continue;   // like the first
        if (p.dx) p.slab_bytes = std::max<uint64_t>(p.slab_bytes, inner_gemm_slab_bytes(ctx, dx_gemm(d, p, 256, 256, 256, r0, n)));
    }
    p.slabs = take(p.slab_bytes);
    p.total = std::max<uint64_t>(off, 256);
    return p;
}

// Sizes that int and the row and tile counters hold.
bool sizes_ok(const t0b_linear_loss& d) { return d.rows <= 0x7fffff00u && d.dim <= 0x7fffff00u && d.vocab <= 0x7fffff00u; }

int32_t check_desc(t0b_ctx* ctx, const char* what, const t0b_linear_loss& d) {
    auto bad = [&](const char* msg) { return set_error(ctx, T0B_ERR_INVALID, "%s: %s", what, msg); };
    if (!d.x || !d.w) return bad("null x or w");
    if (d.dim == 0 || d.vocab == 0) return bad("an empty head");
    if (!sizes_ok(d)) return bad("a size is over 2^31");
    if (!d.losses && !d.lse && !d.dx && !d.dw) return bad("no output is asked for");
    if (d.ldx < d.dim || d.ldw < (d.trans_w ? d.dim : d.vocab) || (d.dx && d.lddx < d.dim) || (d.dw && d.lddw < (d.trans_w ? d.dim : d.vocab)))
        return bad("a pitch is smaller than its row");
    if (d.x_dtype != T0B_OUT_F32 && d.x_dtype != T0B_OUT_BF16) return bad("unknown x_dtype");
    if ((d.dx && d.dx_dtype != T0B_OUT_F32 && d.dx_dtype != T0B_OUT_BF16) || (d.dw && d.dw_dtype != T0B_OUT_F32 && d.dw_dtype != T0B_OUT_BF16))
        return bad("unknown gradient type");
    if (!std::isfinite(d.scale)) return bad("scale is not finite");
    const uint64_t xe = d.x_dtype == T0B_OUT_BF16 ? 2 : 4, dxe = d.dx_dtype == T0B_OUT_BF16 ? 2 : 4, dwe = d.dw_dtype == T0B_OUT_BF16 ? 2 : 4;
    if (d.x % xe || d.w % 2 || (d.dx && d.dx % dxe) || (d.dw && d.dw % dwe) || d.losses % 4 || d.lse % 4 || d.row_weights % 4)
        return bad("a pointer is not aligned to its element");
    const uint64_t wr = d.trans_w ? d.vocab : d.dim, wc = d.trans_w ? d.dim : d.vocab;
    if (d.rows == 0) return check_fits(ctx, what, {{"dw", d.dw, span_bytes(wr, d.lddw, wc, dwe)}});   // becomes zeros
    return check_fits(ctx, what, {{"x", d.x, span_bytes(d.rows, d.ldx, d.dim, xe)}, {"w", d.w, span_bytes(wr, d.ldw, wc, 2)},
                                  {"dx", d.dx, span_bytes(d.rows, d.lddx, d.dim, dxe)}, {"dw", d.dw, span_bytes(wr, d.lddw, wc, dwe)},
                                  {"losses", d.losses, d.rows * 4ull}, {"lse", d.lse, d.rows * 4ull}, {"row_weights", d.row_weights, d.rows * 4ull}});
}

// The scratch of a call: the caller's, else the context's, which grows as needed.  A captured call has to bring its own: the
// context's may be replaced by a later, larger call while the graph still refers to it.
int32_t get_scratch(t0b_ctx* ctx, const char* what, const t0b_linear_loss& d, uint64_t need, uint64_t* at) {
    if (d.scratch) {
        if (d.scratch % 256 || d.scratch_bytes < need)
            return set_error(ctx, T0B_ERR_INVALID, "%s: scratch must be 256-byte aligned and hold %llu bytes (got %llu)", what,
                             static_cast<unsigned long long>(need), static_cast<unsigned long long>(d.scratch_bytes));
        *at = d.scratch;
        return check_fits(ctx, what, {{"scratch", d.scratch, need}});
    }
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    int32_t rc = check_cuda(ctx, cudaStreamIsCapturing(ctx->stream, &st), "cudaStreamIsCapturing");
    if (rc != T0B_OK) return rc;
    if (ctx->capturing || st != cudaStreamCaptureStatusNone)
        return set_error(ctx, T0B_ERR_INVALID, "%s: a captured call needs a scratch of its own (%llu bytes)", what, static_cast<unsigned long long>(need));
    if (ctx->loss_ws_bytes < need) {
        const uint64_t old = ctx->loss_ws;
        ctx->loss_ws = 0;
        ctx->loss_ws_bytes = 0;
        if (old) {
            rc = t0b_free(ctx, old);   // waits for the stream
            if (rc != T0B_OK) return rc;
        }
        rc = t0b_alloc(ctx, need, &ctx->loss_ws);
        if (rc != T0B_OK) return rc;
        ctx->loss_ws_bytes = need;
    }
    *at = ctx->loss_ws;
    return T0B_OK;
}

uint32_t lin_blocks(t0b_ctx* ctx, uint64_t items) {
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>((items + 255) / 256, static_cast<uint64_t>(ctx->num_sms) * 8)));
}

struct Teacher { uint64_t ids, logits, ldk; uint32_t topk; };   // cross entropy: ids = targets, topk = 1, logits = 0

int32_t run_linear_loss(t0b_ctx* ctx, const char* what, const t0b_linear_loss& d, const Teacher& te, float temperature, int32_t async) {
    const uint64_t dwe = d.dw_dtype == T0B_OUT_BF16 ? 2 : 4;
    if (d.rows == 0) {
        if (!d.dw) return T0B_OK;
        const uint64_t wr = d.trans_w ? d.vocab : d.dim, wc = d.trans_w ? d.dim : d.vocab;
        const bool dense = wr == 1 || d.lddw == wc;
        const uint64_t pitch = d.lddw * dwe, run = dense ? wr * wc * dwe : wc * dwe;
        int32_t rc = T0B_OK;
        if (dense || pitch > 0x7fffffffull) {   // the 2-D form ends at pitches of 2 GiB
            for (uint64_t r = 0; r < (dense ? 1 : wr) && rc == T0B_OK; ++r)
                rc = check_cuda(ctx, cudaMemsetAsync(reinterpret_cast<void*>(d.dw + r * pitch), 0, run, ctx->stream), "cudaMemsetAsync(dw)");
        } else {
            rc = check_cuda(ctx, cudaMemset2DAsync(reinterpret_cast<void*>(d.dw), pitch, 0, run, wr, ctx->stream), "cudaMemset2DAsync(dw)");
        }
        return rc != T0B_OK ? rc : finish(ctx, async, what, 0);
    }
    const bool teacher = te.logits != 0;
    Plan p = make_plan(ctx, d, te.topk, teacher);
    if (d.scratch && d.scratch_bytes < p.total && d.scratch_bytes >= p.slabs) {
        // Sized before a t0b_tune that wants more slabs: the product that does not fit them is not split.
        p.slab_bytes = d.scratch_bytes - p.slabs;
        p.total = d.scratch_bytes;
    }
    uint64_t base = 0;
    int32_t rc = get_scratch(ctx, what, d, p.total, &base);
    if (rc != T0B_OK) return rc;
    const float c = 1.4426950408889634f / temperature, inv_t = 1.0f / temperature;
    int launched = 0;

    const uint64_t x = p.copy_x ? base + p.x : d.x, w = p.copy_w ? base + p.w : d.w;
    __nv_bfloat16* xg = reinterpret_cast<__nv_bfloat16*>(base + p.x);
    __nv_bfloat16* x_out = p.copy_x && !p.gather ? xg : nullptr;
    uint32_t* row_of = p.gather ? reinterpret_cast<uint32_t*>(base + p.row_of) : nullptr;
    uint32_t* place_of = reinterpret_cast<uint32_t*>(base + p.place_of);
    int* count = p.gather ? reinterpret_cast<int*>(base + p.count) : nullptr;
    float* losses = reinterpret_cast<float*>(d.losses);
    float* lse = reinterpret_cast<float*>(d.lse);
    const bool x16 = d.x_dtype == T0B_OUT_BF16;
    const __nv_bfloat16* xb = reinterpret_cast<const __nv_bfloat16*>(d.x);
    const float* xf = reinterpret_cast<const float*>(d.x);
    if (teacher) {
        uint32_t P = 32;
        while (P < te.topk) P *= 2;
        const uint32_t ny = std::max(1u, 128u / P);
        auto words = [&](auto kernel, auto* xp) {
            launch(ctx, kernel, dim3((d.rows + ny - 1) / ny), dim3(P, ny), static_cast<size_t>(P) * ny * 12, reinterpret_cast<const uint32_t*>(te.ids),
                   reinterpret_cast<const float*>(te.logits), te.ldk, d.rows, te.topk, d.vocab, inv_t, reinterpret_cast<uint32_t*>(base + p.ids),
                   reinterpret_cast<float*>(base + p.q), reinterpret_cast<float*>(base + p.entropy), reinterpret_cast<uint32_t*>(base + p.live),
                   ctx->status_dev, xp, d.ldx, x_out, static_cast<uint32_t>(p.ldx), d.dim);
        };
        if (x16) words(teacher_words_kernel<__nv_bfloat16>, xb);
        else words(teacher_words_kernel<float>, xf);
        ++launched;
    } else if (x_out) {
        const uint32_t blocks = lin_blocks(ctx, d.rows * (p.ldx / 8));
        const uint32_t* targets = reinterpret_cast<const uint32_t*>(te.ids);
        if (x16) launch(ctx, pack_rows_kernel<__nv_bfloat16>, blocks, 256, 0, xb, d.ldx, x_out, static_cast<uint32_t>(p.ldx), d.rows, d.dim, targets, d.vocab);
        else launch(ctx, pack_rows_kernel<float>, blocks, 256, 0, xf, d.ldx, x_out, static_cast<uint32_t>(p.ldx), d.rows, d.dim, targets, d.vocab);
        ++launched;
    }
    if (p.gather) {
        launch(ctx, live_rows_kernel, 1, 1024, 0, teacher ? nullptr : reinterpret_cast<const uint32_t*>(te.ids),
               teacher ? reinterpret_cast<const uint32_t*>(base + p.live) : nullptr, d.vocab, d.rows, row_of, place_of, count, losses, lse, ctx->status_dev);
        const uint32_t blocks = lin_blocks(ctx, d.rows * (p.ldx / 8));
        if (x16) launch(ctx, gather_rows_kernel<__nv_bfloat16>, blocks, 256, 0, xb, d.ldx, xg, static_cast<uint32_t>(p.ldx), d.rows, d.dim, row_of, count);
        else launch(ctx, gather_rows_kernel<float>, blocks, 256, 0, xf, d.ldx, xg, static_cast<uint32_t>(p.ldx), d.rows, d.dim, row_of, count);
        launched += 2;
    }
    if (p.copy_w) {
        const uint32_t groups = static_cast<uint32_t>(p.ldw / 8), high = groups <= 32 ? 8 : (groups <= 128 ? 2 : 1), wide = 256 / high;
        auto copy = high == 8 ? pack_shifted_kernel<8> : (high == 2 ? pack_shifted_kernel<2> : pack_shifted_kernel<1>);
        launch(ctx, copy, dim3((groups + wide - 1) / wide, static_cast<uint32_t>(std::min<uint64_t>((p.w_rows + high - 1) / high, 65535))), dim3(wide, high), 0,
               reinterpret_cast<const __nv_bfloat16*>(d.w), d.ldw, reinterpret_cast<__nv_bfloat16*>(base + p.w), static_cast<uint32_t>(p.ldw),
               static_cast<uint32_t>(p.w_rows), static_cast<uint32_t>(p.w_cols));
        ++launched;
    }
    rc = check_cuda(ctx, cudaGetLastError(), what);   // what follows takes row numbers from these kernels
    if (rc != T0B_OK) return rc;
    uint32_t part_shift = 0;
    while ((1u << part_shift) < p.head.part_cols) ++part_shift;
    for (uint32_t r0 = 0; r0 < d.rows; r0 += p.piece) {
        const uint32_t n = std::min(p.piece, d.rows - r0);
        Targets tg{};
        tg.ids = reinterpret_cast<const uint32_t*>(teacher ? base + p.ids : te.ids);
        if (teacher) {
            tg.q = reinterpret_cast<const float*>(base + p.q);
            tg.entropy = reinterpret_cast<const float*>(base + p.entropy);
            tg.live = reinterpret_cast<const uint32_t*>(base + p.live);
        }
        tg.z_sel = reinterpret_cast<const float*>(base + p.z_sel);
        tg.n_ids = te.topk;
        tg.vocab = d.vocab;
        tg.row_of = row_of;
        tg.count = count;
        tg.row0 = r0;
        HeadGemm hg{};
        hg.plan = p.head;
        hg.ldx = p.copy_x ? p.ldx : d.ldx; hg.ldw = p.ldw;
        hg.x = x + static_cast<uint64_t>(r0) * hg.ldx * 2;
        hg.w = w;
        hg.rows = n; hg.dim = d.dim; hg.vocab = d.vocab; hg.trans_w = d.trans_w;
        hg.c = c;
        hg.part = base + p.part; hg.part_ld = p.part_ld;
        hg.ids = reinterpret_cast<uint64_t>(tg.ids) + (row_of ? 0 : static_cast<uint64_t>(r0) * te.topk * 4);
        hg.row_of = row_of ? reinterpret_cast<uint64_t>(row_of + r0) : 0;
        hg.dyn_rows = reinterpret_cast<uint64_t>(count);
        hg.dyn_off = static_cast<int>(r0);
        hg.z_sel = reinterpret_cast<uint64_t>(tg.z_sel);
        hg.n_ids = te.topk;
        hg.u = p.grads ? base + p.u : 0;
        hg.ldu = p.ldu;
        rc = head_gemm(ctx, hg);
        if (rc != T0B_OK) return rc;
        float2* stats = reinterpret_cast<float2*>(base + p.stats);
        if (!p.join_in_dz) {
            launch(ctx, join_parts_kernel, (n + 31) / 32, 1024, 0, reinterpret_cast<const float2*>(base + p.part), p.part_ld, p.parts, n, c, inv_t, tg, stats,
                   losses, lse, ctx->status_dev);
            ++launched;
        }
        if (!p.grads) continue;
        const JoinParams jp{p.parts, inv_t, losses, lse, ctx->status_dev};
        const CopyParams cp{p.late_x ? xb : nullptr, d.ldx, p.dw ? xg : nullptr, static_cast<uint32_t>(p.ldx), d.dim};
        for (uint32_t y0 = 0; y0 < n; y0 += 65535u) {   // gridDim.y is limited to 65535
            launch(ctx, p.join_in_dz ? dz_kernel<true> : dz_kernel<false>, dim3(static_cast<uint32_t>((p.ldu + kGradCols - 1) / kGradCols), std::min(65535u, n - y0)),
                   256, 0, reinterpret_cast<__half*>(base + p.u), p.ldu, n, y0, reinterpret_cast<const float2*>(base + p.part), p.part_ld, part_shift, stats,
                   reinterpret_cast<const float*>(d.row_weights), d.scale / temperature, c, tg, jp, cp);
            ++launched;
        }
        rc = check_cuda(ctx, cudaGetLastError(), what);
        if (rc != T0B_OK) return rc;
        if (p.dx) {
            InnerGemm g = dx_gemm(d, p, base + p.u, w, base, r0, n);
            g.slabs = base + p.slabs;
            g.slab_bytes = p.slab_bytes;
            rc = inner_gemm(ctx, g);
            if (rc != T0B_OK) return rc;
        }
        if (p.dw) {
            InnerGemm g = dw_gemm(d, p, base + p.u, p.late_x ? base + p.x : x, base, r0, n);
            // Both gradient products need dz alone, so after a short first one of few rows the second need not wait for it and
            // fills the SMs that it leaves (128 x 1024 -> 32000: 95 -> 84 us a step).  Longer ones run one after the other:
            // side by side they compete for L2 (4096 x 4096 -> 128000: 11.3 -> 11.6 ms, 5806 x 448 -> 6400: 163 -> 172 us).
            g.late_wait = p.dx && n <= 1024 && 2.0 * n * d.dim * d.vocab < 1e11;
            g.slabs = base + p.slabs;
            g.slab_bytes = p.slab_bytes;
            rc = inner_gemm(ctx, g);
            if (rc != T0B_OK) return rc;
        }
    }
    if (p.gather && p.dx) {
        const bool dx16 = d.dx_dtype == T0B_OUT_BF16;
        const uint32_t blocks = lin_blocks(ctx, d.rows * (p.ld_dxg / (dx16 ? 8 : 4)));
        if (dx16)
            launch(ctx, spread_rows_kernel<uint16_t>, blocks, 256, 0, reinterpret_cast<const uint16_t*>(base + p.dxg), static_cast<uint32_t>(p.ld_dxg),
                   reinterpret_cast<uint16_t*>(d.dx), d.lddx, d.rows, d.dim, place_of);
        else
            launch(ctx, spread_rows_kernel<float>, blocks, 256, 0, reinterpret_cast<const float*>(base + p.dxg), static_cast<uint32_t>(p.ld_dxg),
                   reinterpret_cast<float*>(d.dx), d.lddx, d.rows, d.dim, place_of);
        ++launched;
    }
    if (p.acc_dw) {
        launch(ctx, round_rows_kernel, lin_blocks(ctx, p.w_rows * ((p.w_cols + 7) / 8)), 256, 0,
            reinterpret_cast<const float*>(base + p.acc), static_cast<uint32_t>(p.ld_acc), reinterpret_cast<__nv_bfloat16*>(d.dw), d.lddw,
            static_cast<uint32_t>(p.w_rows), static_cast<uint32_t>(p.w_cols));
        ++launched;
    }
    return finish(ctx, async, what, launched);
}

}  // namespace

extern "C" {

size_t t0b_linear_loss_scratch_bytes(t0b_ctx* ctx, const t0b_linear_loss* loss, uint32_t topk) try {
    if (!ctx || !loss || loss->rows == 0 || loss->dim == 0 || loss->vocab == 0 || !sizes_ok(*loss) || topk > T0B_MAX_TOPK) return 0;
    if (span_bytes(loss->vocab, loss->dim, loss->dim, 4) > kMaxSpan) return 0;   // a head that no call takes
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    if (precheck(ctx) != T0B_OK) return 0;
    return make_plan(ctx, *loss, std::max(1u, topk), topk > 0).total;
} catch (...) {
    return 0;
}

// No C++ exception (the host's memory running out) leaves a C entry.
int32_t t0b_linear_ce(t0b_ctx* ctx, const t0b_linear_loss* loss, uint64_t targets, int32_t async) try {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (!loss || !targets || targets % 4) return set_error(ctx, T0B_ERR_INVALID, "linear_ce: null or misaligned pointer");
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    rc = check_desc(ctx, "linear_ce", *loss);
    if (rc == T0B_OK) rc = check_fits(ctx, "linear_ce", {{"targets", targets, loss->rows * 4ull}});
    if (rc != T0B_OK) return rc;
    return run_linear_loss(ctx, "linear_ce", *loss, Teacher{targets, 0, 1, 1}, 1.0f, async);
} catch (...) {
    return T0B_ERR_NOMEM;
}

int32_t t0b_linear_topk_distill(t0b_ctx* ctx, const t0b_linear_loss* loss, uint64_t ids, uint64_t teacher, uint32_t topk, uint64_t ldk,
                                float temperature, int32_t async) try {
    int32_t rc = precheck(ctx, async);
    if (rc != T0B_OK) return rc;
    if (!loss || !ids || !teacher || ids % 4 || teacher % 4) return set_error(ctx, T0B_ERR_INVALID, "linear_topk_distill: null or misaligned pointer");
    if (topk == 0 || topk > T0B_MAX_TOPK || ldk < topk)
        return set_error(ctx, T0B_ERR_INVALID, "linear_topk_distill: topk %u is outside 1..%d, or its pitch %llu is smaller", topk, T0B_MAX_TOPK,
                         static_cast<unsigned long long>(ldk));
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(1.4426950408889634f / temperature))
        return set_error(ctx, T0B_ERR_INVALID, "linear_topk_distill: temperature %g must be positive and finite, and so must its inverse", temperature);
    if (!std::isfinite(loss->scale / temperature))
        return set_error(ctx, T0B_ERR_INVALID, "linear_topk_distill: scale %g over temperature %g is not finite", loss->scale, temperature);
    std::lock_guard<std::recursive_mutex> lk(ctx->mu);
    rc = check_desc(ctx, "linear_topk_distill", *loss);
    if (rc == T0B_OK && loss->rows > 0)
        rc = check_fits(ctx, "linear_topk_distill", {{"ids", ids, span_bytes(loss->rows, ldk, topk, 4)}, {"teacher", teacher, span_bytes(loss->rows, ldk, topk, 4)}});
    if (rc != T0B_OK) return rc;
    return run_linear_loss(ctx, "linear_topk_distill", *loss, Teacher{ids, teacher, ldk, topk}, temperature, async);
} catch (...) {
    return T0B_ERR_NOMEM;
}

}  // extern "C"
