// Internal declarations shared by the translation units of libt0b200.so.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <map>
#include <mutex>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/t0b200.h"

struct t0b_ctx {
    int device = 0;
    int num_sms = 148;
    bool pdl = true;            // launch GEMMs with programmatic stream serialization (T0B_PDL=0 turns it off)
    int raster_group = 0;       // > 0: rasterisation group width for every GEMM (T0B_RASTER_GROUP, for measurements); 0 = chosen per shape
    bool cluster_splitk = true; // split-K of single-CTA tiles runs as thread-block clusters (T0B_CLUSTER_SPLITK=0: slabs + reduce kernel)
    std::string force_config;   // T0_FORCE_CONFIG=<preset name>: the tile every GEMM without an explicit config runs
    bool dump_config = false;   // T0_DUMP_CONFIG=1: print the config and the kernel variant of each new GEMM shape to stderr
    std::map<std::string, int> dumped;
    unsigned wait_hint_ns = 20000;   // T0B_WAIT_HINT_NS: how long an epilogue warp may sleep in hardware per poll of its accumulator barrier
    // Timeline build: where the stamps of the next GEMM launches go (t0b_trace_set); unused in the regular build.
    uint64_t trace_buf = 0;
    uint32_t trace_slots = 0, trace_next = 0;
    int sm_limit = 0;           // > 0: the persistent GEMM kernels occupy at most this many SMs
    cudaStream_t own_stream = nullptr;
    cudaStream_t stream = nullptr;
    cudaEvent_t default_event = nullptr;   // the default stream's work that a synchronous call waits for
    bool default_order = true;             // T0B_DEFAULT_STREAM_ORDER=0: synchronous calls leave the default stream alone
    std::recursive_mutex mu;
    std::string last_error;
    bool poisoned = false;
    // Device status word: pinned host memory mapped into the device, so a kernel can report that one of its
    // bounded waits ran out without any copy.
    int* status_host = nullptr;
    int* status_dev = nullptr;
    unsigned long long wait_limit_ns = 2000000000ull;
    int last_status = 0;        // the code most recently taken from the status word (kept for t0b_device_status)
    // Buffer pool keyed by 4 KiB-rounded size.
    std::multimap<size_t, void*> pool_free;
    std::unordered_map<void*, size_t> live;
    uint64_t pool_cached = 0, pool_hits = 0, pool_misses = 0;
    // Grow-only split-K workspace.
    void* ws = nullptr;
    size_t ws_bytes = 0;
    // Grow-only workspace of the vocabulary losses (from the pool; never used by a call that is being captured).
    uint64_t loss_ws = 0;
    size_t loss_ws_bytes = 0;
    // bf16 copies of f32 weight buffers, by caller-chosen tensor id (GpuRuntime::bf16_cache, src/ignis/gpu_context.rs:392-432).
    struct Bf16Entry { uint64_t ptr; size_t n; };
    std::unordered_map<uint64_t, Bf16Entry> bf16_cache;
    uint64_t bf16_conversions = 0, bf16_hits = 0;
    // Tensor-map cache.
    struct TmapKey {
        uint64_t ptr, d0, d1, ld;
        uint32_t b0, b1, elem;
        bool operator==(const TmapKey& o) const {
            return ptr == o.ptr && d0 == o.d0 && d1 == o.d1 && ld == o.ld && b0 == o.b0 && b1 == o.b1 && elem == o.elem;
        }
    };
    struct TmapHash {
        size_t operator()(const TmapKey& k) const {
            uint64_t h = k.ptr * 0x9E3779B97F4A7C15ull;
            h ^= (k.d0 + 0x9E3779B97F4A7C15ull + (h << 6) + (h >> 2));
            h ^= (k.d1 + 0x9E3779B97F4A7C15ull + (h << 6) + (h >> 2));
            h ^= (k.ld + 0x9E3779B97F4A7C15ull + (h << 6) + (h >> 2));
            h ^= ((static_cast<uint64_t>(k.b0) << 32 | k.b1) + (h << 6) + (h >> 2));
            h ^= (k.elem + 0x9E3779B97F4A7C15ull + (h << 6) + (h >> 2));
            return static_cast<size_t>(h);
        }
    };
    std::unordered_map<TmapKey, CUtensorMap, TmapHash> tmaps;
    // Graph capture.
    bool capturing = false;
    std::unordered_map<uint64_t, cudaGraphExec_t> graphs;
    uint64_t next_graph = 1;
    uint64_t launches = 0;
    std::string autotune_dir;   // empty: the disk cache is not consulted
    // Copy streams of the host-buffer GEMM (created on first use).
    cudaStream_t h2d_stream = nullptr, d2h_stream = nullptr;
    bool d2h_pending = false;   // an asynchronous read-back was queued since the last t0b_sync
    cudaStream_t p2p_stream = nullptr;   // device-to-device / peer copies that run beside the compute stream
    bool p2p_pending = false;
};

namespace t0b {

int32_t set_error(t0b_ctx* ctx, int32_t code, const char* fmt, ...);
int32_t check_cuda(t0b_ctx* ctx, cudaError_t e, const char* what);
// Status-word code of a kernel that met an index outside its table (the access is skipped); 101..105 are the GEMM's
// bounded waits.
constexpr int kDevBadIndex = 110;
// Buffers that start one of the runtime's own allocations must fit in it: an undersized one is reported instead of faulting
// on the device.  (Pointers from elsewhere, or into the middle of a buffer, are not known; null ones are skipped.)  No buffer
// spans more than kMaxSpan bytes: a pitch that says so is refused, whoever allocated.
struct Extent { const char* name; uint64_t ptr; uint64_t bytes; };
constexpr uint64_t kMaxSpan = 1ull << 47;
// From the first to the last byte of `rows` (at least one) rows of `cols` elements at a pitch of `ld`; more than kMaxSpan where
// the true number does not fit 64 bits.
inline uint64_t span_bytes(uint64_t rows, uint64_t ld, uint64_t cols, uint64_t elem) {
    const unsigned __int128 n = (static_cast<unsigned __int128>(rows - 1) * ld + cols) * elem;
    return n > kMaxSpan ? kMaxSpan + 1 : static_cast<uint64_t>(n);
}
int32_t check_fits(t0b_ctx* ctx, const char* what, std::initializer_list<Extent> extents);
int32_t precheck(t0b_ctx* ctx, int32_t async = 1);   // null / poisoned checks, sets the device; a synchronous call waits for the default stream
// Launch-error check (+ sync and status-word check when !async). `count` kernels are added to the launch counter.
int32_t finish(t0b_ctx* ctx, int32_t async, const char* what, int count = 1);
// Read the status word; a non-zero code is moved to ctx->last_status and the word is cleared, so one failed kernel is
// reported by one call and does not fail the calls after it.
int take_device_status(t0b_ctx* ctx);

// Host-side GemmConfig logic (t0b_gemm_gen.cpp).
void default_b200_config(uint32_t m, uint32_t k, uint32_t n, int num_sms, t0b_gemm_config* out);

// Measured configs (t0b_gemm_gen.cpp): results of t0b_tune in this process, then the table shipped with the library.
bool tuned_lookup(uint32_t m, uint32_t n, uint32_t k, int trans_a, int trans_b, int out_bf16, t0b_gemm_config* out, int* source);
void tuned_remember(uint32_t m, uint32_t n, uint32_t k, int trans_a, int trans_b, int out_bf16, const t0b_gemm_config& cfg);
void tuned_forget(uint32_t m, uint32_t n, uint32_t k);

struct PlanInput {
    uint32_t m, n, k;
    int trans_a, trans_b;
    uint64_t lda, ldb;
    uint64_t a_ptr, b_ptr;
    int num_sms;
};
void resolve_plan(const t0b_gemm_config* cfg, const PlanInput& in, t0b_gemm_plan* out);
// Products inside other operators (t0b_gemm.cu): the same kernels and choice of tile as t0b_gemm.  Operands are 16-byte
// aligned with pitches of whole 16 bytes.  `slabs` holds inner_gemm_slab_bytes() bytes for a split-K through global memory.
struct InnerGemm {
    int trans_a, trans_b;
    uint64_t a, b, c;
    uint32_t m, n, k;
    uint64_t lda, ldb, ldc;
    int out_bf16;
    bool accumulate;   // C += A*B, f32
    bool head_grad;    // the head's gradient: its own choice of tile, never split
    uint64_t slabs;
    size_t slab_bytes;
    uint64_t dyn_rows;   // device int, or 0: m (dyn_k: k) is at most *dyn_rows - dyn_off
    int dyn_off, dyn_k;
    bool late_wait;      // runs beside the product launched just before it, which had the same operands complete (GemmParams)
};
size_t inner_gemm_slab_bytes(t0b_ctx* ctx, const InnerGemm& d);
int32_t inner_gemm(t0b_ctx* ctx, const InnerGemm& d);

// The product x * head whose epilogue leaves softmax statistics instead of logits (HeadParams, gemm_sm100.cuh).
constexpr float kHeadUScale = 32768.0f;   // of the exponentials that it leaves in fp16
struct HeadPlan { uint32_t bm, bn, cta_group, part_cols; };
HeadPlan head_plan(t0b_ctx* ctx, uint32_t rows, uint32_t vocab, uint32_t dim);
struct HeadGemm {
    HeadPlan plan;
    uint64_t x, w;               // bf16; w [dim, vocab], or [vocab, dim] with trans_w
    uint64_t ldx, ldw;
    uint32_t rows, dim, vocab;
    int trans_w;
    float c;                     // log2(e) / temperature
    uint64_t part, part_ld;      // float2 [ceil(vocab / part_cols)][part_ld]
    uint64_t ids, z_sel;         // u32 / f32 [rows][n_ids]
    uint32_t n_ids;
    uint64_t row_of;             // u32[rows]: the row of ids that belongs to a row of x; 0 = the same
    uint64_t dyn_rows;           // device int, or 0: rows is at most *dyn_rows - dyn_off
    int dyn_off;
    uint64_t u, ldu;             // fp16 [rows][ldu], ldu a multiple of 8; 0 = statistics alone
};
int32_t head_gemm(t0b_ctx* ctx, const HeadGemm& d);

// tile_ir front end (t0b_tile_ir.cpp): spec validation and the offsets of the epilogue arguments in its kernarg blob.
bool tile_spec_valid(const t0b_tile_gemm* spec);
size_t tile_kernarg_layout(const t0b_tile_gemm* spec, size_t* bias_off, size_t* scale_off, size_t* clamp_off);

}  // namespace t0b
