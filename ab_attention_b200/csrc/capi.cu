// extern "C" boundary of libabx (declared in include/abx.h).
//
// Validates every argument on the host, lays out the caller-owned workspace,
// and launches the kernels on the caller's stream. No allocation, no host
// synchronisation (except abx_device_status, which reads the error word).
#include <cuda.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "chunk.cuh"
#include "common.cuh"
#include "ibcs.cuh"
#include "rotary.cuh"
#include "tcgen05.cuh"
#include "tma_host.cuh"

namespace abx {

__device__ int g_device_error = 0;

int* device_error_word() {
    void* ptr = nullptr;
    if (cudaGetSymbolAddress(&ptr, g_device_error) != cudaSuccess) return nullptr;
    return static_cast<int*>(ptr);
}

// Two warps wait, bounded by limit_cycles, on an mbarrier that nothing arrives
// at: warp 0 with the library's polling wait, warp 1 with its suspending wait
// (the form the prefill kernels use). Both give up, each on its own abort flag,
// and the kernel records ABX_ERR_DEVICE_TIMEOUT only when both did, exercising
// both timeout paths without a fault.
__global__ void wait_selftest_kernel(uint64_t limit_cycles, int* error) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ int abort_flag[2];
    __shared__ int gave_up[2];
    const int w = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        abort_flag[0] = abort_flag[1] = 0;
        tc::mbar_init(smem_addr(&bar), 1);
        tc::mbar_init_fence();
    }
    __syncthreads();
    const bool ok = w == 0 ? tc::mbar_wait_warp(smem_addr(&bar), 0, &abort_flag[0], limit_cycles)
                           : tc::mbar_wait_warp_suspend(smem_addr(&bar), 0, &abort_flag[1], limit_cycles);
    if ((threadIdx.x & 31) == 0) gave_up[w] = !ok;
    __syncthreads();
    if (threadIdx.x == 0 && gave_up[0] && gave_up[1]) raise_device_error(error, ABX_ERR_DEVICE_TIMEOUT);
}

}  // namespace abx

namespace {

thread_local char g_last_error[512] = "";

int fail(int status, const char* fmt, ...) {
    va_list args;
    va_start(args, fmt);
    vsnprintf(g_last_error, sizeof(g_last_error), fmt, args);
    va_end(args);
    return status;
}

int check_cuda(cudaError_t err, const char* what) {
    if (err == cudaSuccess) return ABX_OK;
    return fail(ABX_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

// A driver API call reached through the runtime's entry-point table (no libcuda link).
template <class Fn>
Fn driver_entry(const char* name) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult status;
    if (cudaGetDriverEntryPoint(name, &ptr, cudaEnableDefault, &status) != cudaSuccess ||
        status != cudaDriverEntryPointSuccess)
        return nullptr;
    return reinterpret_cast<Fn>(ptr);
}

constexpr size_t kAlign = 256;
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Workspace of the IBCS stages for (bh, seq).
struct IbcsLayout {
    int64_t qb, rows, fine, ld;
    size_t scaled, populations, pooled, lse, lse_max, lse_den, total;
};

IbcsLayout ibcs_layout(int64_t bh, int64_t seq) {
    IbcsLayout l{};
    l.qb = abx::ceil_div(seq, abx::kQueryBlock);
    l.rows = bh * l.qb;
    l.fine = seq / abx::kKv4;
    l.ld = (l.fine + 7) / 8 * 8;
    size_t off = 0;
    l.scaled = off;
    off = align_up(off + static_cast<size_t>(l.rows) * abx::kCentroids * abx::kHeadDim * 2);
    l.populations = off;
    off = align_up(off + static_cast<size_t>(l.rows) * abx::kCentroids * 4);
    l.pooled = off;
    off = align_up(off + static_cast<size_t>(bh) * l.fine * abx::kReps * abx::kHeadDim * 2);
    l.lse = off;
    off = align_up(off + static_cast<size_t>(l.rows) * abx::kCentroids * l.ld * 2);
    l.lse_max = off;
    off = align_up(off + static_cast<size_t>(l.rows) * abx::kCentroids * 4);
    l.lse_den = off;
    off = align_up(off + static_cast<size_t>(l.rows) * abx::kCentroids * 4);
    // No block-score array: abx_build_plan's SIP evaluates the mixture from the
    // LSE rows, and abx_ibcs_scores writes the caller's scores.
    l.total = off;
    return l;
}

int check_qk_shape(int64_t bh, int64_t seq) {
    if (bh <= 0) return fail(ABX_ERR_INVALID_ARGUMENT, "batch*heads must be positive (got %lld)", (long long)bh);
    if (seq <= 0 || seq % abx::kKv4 != 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "sequence length must be a positive multiple of 4 (got %lld)", (long long)seq);
    const int64_t fine = seq / abx::kKv4;
    if (fine > abx::kMaxFineBlocks)
        return fail(ABX_ERR_UNSUPPORTED, "KV4 block count must be in [1, 32768] (got %lld)", (long long)fine);
    if (bh * abx::ceil_div(seq, abx::kQueryBlock) > 0x7fffffffLL)
        return fail(ABX_ERR_UNSUPPORTED, "too many query blocks");
    return ABX_OK;
}

int check_sip_shape(int64_t rows, int64_t population, int64_t samples) {
    if (rows <= 0) return fail(ABX_ERR_INVALID_ARGUMENT, "row count must be positive");
    if (samples <= 0 || samples >= population)
        return fail(ABX_ERR_INVALID_ARGUMENT, "sample count must be inside the population (0 < %lld < %lld)",
                    (long long)samples, (long long)population);
    if (population > 0x7fffffffLL) return fail(ABX_ERR_UNSUPPORTED, "population too large");
    const size_t need = abx::sip_smem_bytes(population);
    const int limit = abx::sip_smem_limit();
    if (limit <= 0 || need > static_cast<size_t>(limit))
        return fail(ABX_ERR_UNSUPPORTED, "population exceeds single-block shared memory capacity (%zu > %d bytes)",
                    need, limit);
    return ABX_OK;
}

}  // namespace

extern "C" {

int abx_version(void) { return 1; }

const char* abx_status_string(int status) {
    switch (status) {
        case ABX_OK: return "ok";
        case ABX_ERR_INVALID_ARGUMENT: return "invalid argument";
        case ABX_ERR_UNSUPPORTED: return "unsupported shape";
        case ABX_ERR_WORKSPACE: return "workspace too small or misaligned";
        case ABX_ERR_CUDA: return "CUDA error";
        case ABX_ERR_DEVICE_TIMEOUT: return "device-side wait timed out";
        default: return "unknown status";
    }
}

const char* abx_last_error(void) { return g_last_error; }

int abx_device_status(abx_stream_t stream, int clear, int* status_out) {
    if (status_out == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "status_out is null");
    int value = 0;
    int st = check_cuda(cudaMemcpyFromSymbolAsync(&value, abx::g_device_error, sizeof(int), 0,
                                                  cudaMemcpyDeviceToHost, stream),
                        "read device status");
    if (st) return st;
    st = check_cuda(cudaStreamSynchronize(stream), "synchronize");
    if (st) return st;
    if (clear) {
        const int zero = 0;
        st = check_cuda(cudaMemcpyToSymbolAsync(abx::g_device_error, &zero, sizeof(int), 0,
                                                cudaMemcpyHostToDevice, stream),
                        "clear device status");
        if (st) return st;
        st = check_cuda(cudaStreamSynchronize(stream), "synchronize");
        if (st) return st;
    }
    *status_out = value;
    return ABX_OK;
}

int abx_ibcs_cluster(const void* q, int64_t bh, int64_t seq, void* centroids, void* scaled_centroids,
                     float* populations, int32_t* assignments, abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (q == nullptr || populations == nullptr)
        return fail(ABX_ERR_INVALID_ARGUMENT, "q and populations must be non-null");
    if (!aligned16(q) || (centroids && !aligned16(centroids)) || (scaled_centroids && !aligned16(scaled_centroids)))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q and centroid buffers must be 16-byte aligned");
    return check_cuda(abx::launch_cluster(static_cast<const abx::bf16*>(q), bh, seq,
                                          static_cast<abx::bf16*>(centroids),
                                          static_cast<abx::bf16*>(scaled_centroids), populations,
                                          assignments, stream),
                      "cluster launch");
}

int abx_ibcs_pool(const void* k, int64_t bh, int64_t seq, void* pooled, abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (k == nullptr || pooled == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "k and pooled must be non-null");
    if (!aligned16(k) || !aligned16(pooled)) return fail(ABX_ERR_INVALID_ARGUMENT, "k and pooled must be 16-byte aligned");
    return check_cuda(abx::launch_pool(static_cast<const abx::bf16*>(k), bh, seq, static_cast<abx::bf16*>(pooled), stream),
                      "pool launch");
}

int abx_ibcs_lse(const void* scaled_centroids, const void* pooled, int64_t bh, int64_t qb,
                 int64_t fine_blocks, uint16_t* lse, float* lse_max, float* lse_den, abx_stream_t stream) {
    if (bh <= 0 || qb <= 0 || fine_blocks <= 0 || fine_blocks > abx::kMaxFineBlocks)
        return fail(ABX_ERR_INVALID_ARGUMENT, "bad IBCS LSE shape");
    if (!scaled_centroids || !pooled || !lse || !lse_max || !lse_den)
        return fail(ABX_ERR_INVALID_ARGUMENT, "IBCS LSE buffers must be non-null");
    if (!aligned16(scaled_centroids) || !aligned16(pooled) || !aligned16(lse))
        return fail(ABX_ERR_INVALID_ARGUMENT, "IBCS LSE buffers must be 16-byte aligned");
    return check_cuda(abx::launch_lse(static_cast<const abx::bf16*>(scaled_centroids),
                                      static_cast<const abx::bf16*>(pooled), bh, qb, fine_blocks,
                                      fine_blocks, reinterpret_cast<half*>(lse), lse_max, lse_den, stream),
                      "lse launch");
}

int abx_ibcs_mix(const uint16_t* lse, const float* populations, const float* lse_max, const float* lse_den,
                 int64_t rows, int64_t fine_blocks, float* scores, abx_stream_t stream) {
    if (rows <= 0 || fine_blocks <= 0) return fail(ABX_ERR_INVALID_ARGUMENT, "bad IBCS mix shape");
    if (!lse || !populations || !lse_max || !lse_den || !scores)
        return fail(ABX_ERR_INVALID_ARGUMENT, "IBCS mix buffers must be non-null");
    return check_cuda(abx::launch_mix(reinterpret_cast<const half*>(lse), fine_blocks, populations, lse_max,
                                      lse_den, rows, fine_blocks, scores, stream),
                      "mix launch");
}

int abx_ibcs_workspace_size(int64_t bh, int64_t seq, size_t* bytes) {
    if (bytes == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "bytes is null");
    if (int st = check_qk_shape(bh, seq)) return st;
    *bytes = ibcs_layout(bh, seq).total;
    return ABX_OK;
}

static int run_ibcs_front(const void* q, const void* k, int64_t bh, int64_t seq, void* workspace,
                          size_t workspace_bytes, const IbcsLayout& l, cudaStream_t stream) {
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) % kAlign) != 0)
        return fail(ABX_ERR_WORKSPACE, "workspace must be non-null and 256-byte aligned");
    if (workspace_bytes < l.total)
        return fail(ABX_ERR_WORKSPACE, "workspace too small (%zu < %zu bytes)", workspace_bytes, l.total);
    if (!q || !k || !aligned16(q) || !aligned16(k))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q and k must be non-null and 16-byte aligned");
    char* ws = static_cast<char*>(workspace);
    auto* scaled = reinterpret_cast<abx::bf16*>(ws + l.scaled);
    auto* pops = reinterpret_cast<float*>(ws + l.populations);
    auto* pooled = reinterpret_cast<abx::bf16*>(ws + l.pooled);
    auto* lse = reinterpret_cast<half*>(ws + l.lse);
    auto* mx = reinterpret_cast<float*>(ws + l.lse_max);
    auto* den = reinterpret_cast<float*>(ws + l.lse_den);
    // clustering and key pooling in one launch
    if (int st = check_cuda(abx::launch_cluster(static_cast<const abx::bf16*>(q), bh, seq, nullptr, scaled,
                                                pops, nullptr, stream, static_cast<const abx::bf16*>(k), pooled),
                            "cluster launch"))
        return st;
    return check_cuda(abx::launch_lse(scaled, pooled, bh, l.qb, l.fine, l.ld, lse, mx, den, stream), "lse launch");
}

int abx_ibcs_scores(const void* q, const void* k, int64_t bh, int64_t seq, float* scores, void* workspace,
                    size_t workspace_bytes, abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (scores == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "scores is null");
    const IbcsLayout l = ibcs_layout(bh, seq);
    if (int st = run_ibcs_front(q, k, bh, seq, workspace, workspace_bytes, l, stream)) return st;
    char* ws = static_cast<char*>(workspace);
    return check_cuda(abx::launch_mix(reinterpret_cast<const half*>(ws + l.lse), l.ld,
                                      reinterpret_cast<const float*>(ws + l.populations),
                                      reinterpret_cast<const float*>(ws + l.lse_max),
                                      reinterpret_cast<const float*>(ws + l.lse_den), l.rows, l.fine, scores,
                                      stream),
                      "mix launch");
}

int abx_sip(const float* scores, const float* offsets, int64_t rows, int64_t population, int32_t* ids,
            float* log_weights, int64_t samples, abx_stream_t stream) {
    if (int st = check_sip_shape(rows, population, samples)) return st;
    if (!scores || !offsets || !ids || !log_weights)
        return fail(ABX_ERR_INVALID_ARGUMENT, "SIP buffers must be non-null");
    return check_cuda(abx::launch_sip(scores, offsets, rows, population, ids, log_weights, samples, stream),
                      "sip launch");
}

int abx_build_plan(const void* q, const void* k, int64_t bh, int64_t seq, const float* offsets, int64_t samples,
                   int32_t* ids, float* log_weights, void* workspace, size_t workspace_bytes,
                   abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    const IbcsLayout l = ibcs_layout(bh, seq);
    if (int st = check_sip_shape(l.rows, l.fine, samples)) return st;
    if (!offsets || !ids || !log_weights) return fail(ABX_ERR_INVALID_ARGUMENT, "plan buffers must be non-null");
    if (int st = run_ibcs_front(q, k, bh, seq, workspace, workspace_bytes, l, stream)) return st;
    // SIP evaluates the mixture scores from the LSE rows itself (no score array).
    char* ws = static_cast<char*>(workspace);
    return check_cuda(abx::launch_sip_mixed(reinterpret_cast<const half*>(ws + l.lse), l.ld,
                                            reinterpret_cast<const float*>(ws + l.populations),
                                            reinterpret_cast<const float*>(ws + l.lse_max),
                                            reinterpret_cast<const float*>(ws + l.lse_den), offsets, l.rows, l.fine,
                                            ids, log_weights, samples, stream),
                      "sip launch");
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Allocation-free build_plan: the IBCS scratch lives in a fixed device array.
//
// Some callers cannot call cudaMalloc: a host process whose device memory is
// owned by another allocator (a framework's caching pool, or a serving runtime
// that reserves all memory up front), a plugin host that forbids allocation
// after start-up, or a latency-critical path that cannot afford cudaMalloc's
// implicit device synchronisation. abx_build_plan_static serves them: it needs
// no workspace argument and allocates nothing, using the 256 MiB array below,
// which every GPU that loads libabx holds until the process exits.
// ---------------------------------------------------------------------------
namespace {

constexpr size_t kStaticScratchBytes = size_t(256) << 20;
static __device__ __align__(256) unsigned char g_static_scratch[kStaticScratchBytes];

using PfnCtxGetCurrent = CUresult (*)(CUcontext*);
using PfnCtxGetId = CUresult (*)(CUcontext, unsigned long long*);

// The array's device address per CUDA context, keyed by the context's unique
// id (cuCtxGetId never reuses an id within a process). A host that creates its
// own context on a device, or that resets the device, gets a fresh lookup
// instead of an address that belongs to another or a destroyed context.
struct ScratchSlot {
    unsigned long long context_id;
    void* ptr;
};
constexpr int kScratchSlots = 64;
std::mutex g_static_scratch_mutex;
ScratchSlot g_static_scratch_slots[kScratchSlots] = {};
int g_static_scratch_next = 0;

// Device address of g_static_scratch in the calling thread's current context.
// In host code the array's name is only a host-side stand-in, so the address
// is looked up with cudaGetSymbolAddress (with that device current) once per
// context and cached.
int static_scratch(void** out) {
    static const PfnCtxGetCurrent ctx_get_current = driver_entry<PfnCtxGetCurrent>("cuCtxGetCurrent");
    static const PfnCtxGetId ctx_get_id = driver_entry<PfnCtxGetId>("cuCtxGetId");
    if (ctx_get_current == nullptr || ctx_get_id == nullptr)
        return fail(ABX_ERR_CUDA, "cuCtxGetCurrent / cuCtxGetId unavailable in this driver");
    CUcontext ctx = nullptr;
    if (ctx_get_current(&ctx) != CUDA_SUCCESS || ctx == nullptr) {
        // No context is bound to this thread yet: the symbol lookup initialises
        // the current device's primary context and makes it current.
        void* ptr = nullptr;
        if (int st = check_cuda(cudaGetSymbolAddress(&ptr, g_static_scratch), "cudaGetSymbolAddress(static scratch)"))
            return st;
        if (ctx_get_current(&ctx) != CUDA_SUCCESS || ctx == nullptr)
            return fail(ABX_ERR_CUDA, "no current CUDA context after the symbol lookup");
    }
    unsigned long long id = 0;
    if (ctx_get_id(ctx, &id) != CUDA_SUCCESS) return fail(ABX_ERR_CUDA, "cuCtxGetId failed");
    std::lock_guard<std::mutex> lock(g_static_scratch_mutex);
    for (const ScratchSlot& slot : g_static_scratch_slots) {
        if (slot.ptr != nullptr && slot.context_id == id) {
            *out = slot.ptr;
            return ABX_OK;
        }
    }
    void* ptr = nullptr;
    if (int st = check_cuda(cudaGetSymbolAddress(&ptr, g_static_scratch), "cudaGetSymbolAddress(static scratch)"))
        return st;
    g_static_scratch_slots[g_static_scratch_next] = ScratchSlot{id, ptr};
    g_static_scratch_next = (g_static_scratch_next + 1) % kScratchSlots;
    *out = ptr;
    return ABX_OK;
}

}  // namespace

extern "C" {

size_t abx_static_scratch_bytes(void) { return kStaticScratchBytes; }

int abx_build_plan_static(const void* q, const void* k, int64_t bh, int64_t seq, const float* offsets,
                          int64_t samples, int32_t* ids, float* log_weights, abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    const IbcsLayout one = ibcs_layout(1, seq);
    if (one.total > kStaticScratchBytes)
        return fail(ABX_ERR_WORKSPACE,
                    "abx_build_plan_static: one head of %lld tokens needs %zu bytes of scratch, more than the "
                    "fixed %zu-byte array; use abx_build_plan with a caller workspace",
                    (long long)seq, one.total, kStaticScratchBytes);
    if (int st = check_sip_shape(one.rows, one.fine, samples)) return st;
    if (!q || !k || !offsets || !ids || !log_weights)
        return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, offsets, ids and log_weights must be non-null");
    void* scratch = nullptr;
    if (int st = static_scratch(&scratch)) return st;
    // Heads per pass: as many as the array holds; passes run in stream order.
    int64_t per_pass = 1;
    while (per_pass < bh && ibcs_layout(per_pass + 1, seq).total <= kStaticScratchBytes) ++per_pass;
    const int64_t head_elems = seq * abx::kHeadDim;
    for (int64_t start = 0; start < bh; start += per_pass) {
        const int64_t heads = (bh - start) < per_pass ? (bh - start) : per_pass;
        const int64_t row0 = start * one.qb;
        const int st = abx_build_plan(static_cast<const abx::bf16*>(q) + start * head_elems,
                                      static_cast<const abx::bf16*>(k) + start * head_elems, heads, seq,
                                      offsets + row0, samples, ids + row0 * samples, log_weights + row0 * samples,
                                      scratch, kStaticScratchBytes, stream);
        if (st) return st;
    }
    return ABX_OK;
}

int abx_sparse_prefill(const void* q, const void* k, const void* v, int64_t bh, int64_t seq, const int32_t* ids,
                       const float* log_weights, int64_t samples, const void* text_k, const void* text_v,
                       int64_t text_tokens, void* o, float* lse, abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (!q || !k || !v || !o) return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, v and o must be non-null");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, v and o must be 16-byte aligned");
    if (samples < 0 || samples > seq / abx::kKv4)
        return fail(ABX_ERR_INVALID_ARGUMENT, "samples must be in [0, seq/4] (got %lld)", (long long)samples);
    if (samples > 0 && (ids == nullptr || log_weights == nullptr))
        return fail(ABX_ERR_INVALID_ARGUMENT, "ids and log_weights must be non-null");
    if (text_tokens < 0) return fail(ABX_ERR_INVALID_ARGUMENT, "negative text token count");
    if (text_tokens > 0 && (!text_k || !text_v || !aligned16(text_k) || !aligned16(text_v)))
        return fail(ABX_ERR_INVALID_ARGUMENT, "text_k/text_v must be non-null and 16-byte aligned");
    if (samples + (text_tokens + abx::kKv4 - 1) / abx::kKv4 <= 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "every row needs at least one key block");
    return check_cuda(abx::launch_prefill(static_cast<const abx::bf16*>(q), seq, static_cast<const abx::bf16*>(k),
                                          static_cast<const abx::bf16*>(v), bh, seq, ids, log_weights, samples,
                                          static_cast<const abx::bf16*>(text_k),
                                          static_cast<const abx::bf16*>(text_v), text_tokens,
                                          static_cast<abx::bf16*>(o), lse, stream),
                      "prefill launch");
}

int abx_prefill_workspace_size(int64_t bh, int64_t seq, int64_t samples, int64_t text_tokens, size_t* bytes) {
    if (bytes == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "bytes must be non-null");
    if (int st = check_qk_shape(bh, seq)) return st;
    if (samples < 0 || text_tokens < 0) return fail(ABX_ERR_INVALID_ARGUMENT, "negative sample or text count");
    *bytes = abx::pair_supported(seq, samples, text_tokens) ? abx::pair_workspace_bytes(bh, seq, samples, text_tokens)
                                                             : 0;
    return ABX_OK;
}

}  // extern "C"

namespace {

// Arguments of the paired prefill once the shape is known to pair.
int check_paired(const void* q, const void* k, const void* v, int64_t bh, int64_t seq, const int32_t* ids,
                 const float* log_weights, int64_t samples, const void* text_k, const void* text_v,
                 int64_t text_tokens, const void* o, const void* workspace, size_t workspace_bytes) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (!q || !k || !v || !o) return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, v and o must be non-null");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, v and o must be 16-byte aligned");
    if (samples > seq / abx::kKv4)
        return fail(ABX_ERR_INVALID_ARGUMENT, "samples must be in [0, seq/4] (got %lld)", (long long)samples);
    if (ids == nullptr || log_weights == nullptr)
        return fail(ABX_ERR_INVALID_ARGUMENT, "ids and log_weights must be non-null");
    if (text_tokens > 0 && (!text_k || !text_v || !aligned16(text_k) || !aligned16(text_v)))
        return fail(ABX_ERR_INVALID_ARGUMENT, "text_k/text_v must be non-null and 16-byte aligned");
    if (workspace == nullptr || workspace_bytes < abx::pair_workspace_bytes(bh, seq, samples, text_tokens))
        return fail(ABX_ERR_WORKSPACE, "workspace too small (%zu bytes, need %zu)", workspace_bytes,
                    abx::pair_workspace_bytes(bh, seq, samples, text_tokens));
    return ABX_OK;
}

}  // namespace

extern "C" {

int abx_sparse_prefill_paired(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                              const int32_t* ids, const float* log_weights, int64_t samples, const void* text_k,
                              const void* text_v, int64_t text_tokens, void* o, float* lse, void* workspace,
                              size_t workspace_bytes, abx_stream_t stream) {
    if (samples < 0 || text_tokens < 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "negative sample or text token count");
    if (!abx::pair_supported(seq, samples, text_tokens) || ids == nullptr)
        return abx_sparse_prefill(q, k, v, bh, seq, ids, log_weights, samples, text_k, text_v, text_tokens, o, lse,
                                  stream);
    if (int st = check_paired(q, k, v, bh, seq, ids, log_weights, samples, text_k, text_v, text_tokens, o, workspace,
                              workspace_bytes))
        return st;
    return check_cuda(abx::launch_prefill_pair(static_cast<const abx::bf16*>(q), static_cast<const abx::bf16*>(k),
                                               static_cast<const abx::bf16*>(v), bh, seq, ids, log_weights, samples,
                                               static_cast<const abx::bf16*>(text_k),
                                               static_cast<const abx::bf16*>(text_v), text_tokens,
                                               static_cast<abx::bf16*>(o), lse, workspace, workspace_bytes, stream),
                      "paired prefill launch");
}

int abx_ipc_handle(const void* ptr, void* handle, size_t* offset) {
    if (ptr == nullptr || handle == nullptr || offset == nullptr)
        return fail(ABX_ERR_INVALID_ARGUMENT, "ptr, handle and offset must be non-null");
    using PfnAddressRange = CUresult (*)(CUdeviceptr*, size_t*, CUdeviceptr);
    static const PfnAddressRange address_range = driver_entry<PfnAddressRange>("cuMemGetAddressRange");
    if (address_range == nullptr) return fail(ABX_ERR_CUDA, "cuMemGetAddressRange unavailable in this driver");
    CUdeviceptr base = 0;
    size_t bytes = 0;
    if (address_range(&base, &bytes, reinterpret_cast<CUdeviceptr>(ptr)) != CUDA_SUCCESS)
        return fail(ABX_ERR_INVALID_ARGUMENT, "ptr is not device memory of this process");
    cudaIpcMemHandle_t h;
    if (int st = check_cuda(cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base)), "cudaIpcGetMemHandle")) return st;
    std::memcpy(handle, &h, sizeof(h));
    *offset = static_cast<size_t>(reinterpret_cast<CUdeviceptr>(ptr) - base);
    return ABX_OK;
}

int abx_ipc_open(const void* handle, void** base) {
    if (handle == nullptr || base == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "handle and base must be non-null");
    cudaIpcMemHandle_t h;
    std::memcpy(&h, handle, sizeof(h));
    return check_cuda(cudaIpcOpenMemHandle(base, h, cudaIpcMemLazyEnablePeerAccess), "cudaIpcOpenMemHandle");
}

int abx_ipc_close(void* base) {
    if (base == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "base must be non-null");
    return check_cuda(cudaIpcCloseMemHandle(base), "cudaIpcCloseMemHandle");
}

int abx_peer_copy(void* dst, const void* src, size_t bytes, abx_stream_t stream) {
    if (dst == nullptr || src == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "dst and src must be non-null");
    if (bytes == 0) return ABX_OK;
    return check_cuda(cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDefault, stream), "peer copy");
}

int abx_sparse_prefill_scatter(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                               const int32_t* ids, const float* log_weights, int64_t samples, const void* text_k,
                               const void* text_v, int64_t text_tokens, void* const* outs, int num_outs,
                               int64_t out_head_base, int64_t out_heads, float* lse, void* workspace,
                               size_t workspace_bytes, abx_stream_t stream) {
    if (samples < 0 || text_tokens < 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "negative sample or text token count");
    if (outs == nullptr || num_outs < 1 || num_outs > abx::kMaxScatterOutputs)
        return fail(ABX_ERR_INVALID_ARGUMENT, "between 1 and %d output buffers are needed (got %d)",
                    abx::kMaxScatterOutputs, num_outs);
    abx::bf16* dsts[abx::kMaxScatterOutputs];
    for (int d = 0; d < num_outs; ++d) {
        if (outs[d] == nullptr || !aligned16(outs[d]))
            return fail(ABX_ERR_INVALID_ARGUMENT, "output buffer %d must be non-null and 16-byte aligned", d);
        dsts[d] = static_cast<abx::bf16*>(outs[d]);
    }
    if (out_head_base < 0 || out_heads < out_head_base + bh)
        return fail(ABX_ERR_INVALID_ARGUMENT, "heads [%lld, %lld) lie outside the %lld-head output",
                    (long long)out_head_base, (long long)(out_head_base + bh), (long long)out_heads);
    if (!abx::pair_supported(seq, samples, text_tokens))
        return fail(ABX_ERR_UNSUPPORTED, "this shape cannot be paired (abx_prefill_workspace_size reports 0)");
    if (int st = check_paired(q, k, v, bh, seq, ids, log_weights, samples, text_k, text_v, text_tokens, outs[0],
                              workspace, workspace_bytes))
        return st;
    if (int st = check_cuda(abx::launch_pair_plan(ids, bh, seq, samples, text_tokens, workspace, workspace_bytes,
                                                  stream),
                            "pair plan launch"))
        return st;
    return check_cuda(abx::launch_pair_prefill(static_cast<const abx::bf16*>(q), static_cast<const abx::bf16*>(k),
                                               static_cast<const abx::bf16*>(v), bh, seq, ids, log_weights, samples,
                                               static_cast<const abx::bf16*>(text_k),
                                               static_cast<const abx::bf16*>(text_v), text_tokens, nullptr, lse,
                                               workspace, workspace_bytes, stream, dsts, num_outs, out_head_base),
                      "scatter prefill launch");
}

int abx_pair_plan(const int32_t* ids, int64_t bh, int64_t seq, int64_t samples, int64_t text_tokens, void* workspace,
                  size_t workspace_bytes, abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (samples < 0 || text_tokens < 0) return fail(ABX_ERR_INVALID_ARGUMENT, "negative sample or text token count");
    if (!abx::pair_supported(seq, samples, text_tokens))
        return fail(ABX_ERR_UNSUPPORTED, "this shape cannot be paired (abx_prefill_workspace_size reports 0)");
    if (ids == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "ids must be non-null");
    if (workspace == nullptr || workspace_bytes < abx::pair_workspace_bytes(bh, seq, samples, text_tokens))
        return fail(ABX_ERR_WORKSPACE, "workspace too small (%zu bytes, need %zu)", workspace_bytes,
                    abx::pair_workspace_bytes(bh, seq, samples, text_tokens));
    return check_cuda(abx::launch_pair_plan(ids, bh, seq, samples, text_tokens, workspace, workspace_bytes, stream),
                      "pair plan launch");
}

int abx_sparse_prefill_paired_planned(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                                      const int32_t* ids, const float* log_weights, int64_t samples,
                                      const void* text_k, const void* text_v, int64_t text_tokens, void* o,
                                      float* lse, void* workspace, size_t workspace_bytes, abx_stream_t stream) {
    if (samples < 0 || text_tokens < 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "negative sample or text token count");
    if (!abx::pair_supported(seq, samples, text_tokens))
        return fail(ABX_ERR_UNSUPPORTED, "this shape cannot be paired (abx_prefill_workspace_size reports 0)");
    if (int st = check_paired(q, k, v, bh, seq, ids, log_weights, samples, text_k, text_v, text_tokens, o, workspace,
                              workspace_bytes))
        return st;
    return check_cuda(abx::launch_pair_prefill(static_cast<const abx::bf16*>(q), static_cast<const abx::bf16*>(k),
                                               static_cast<const abx::bf16*>(v), bh, seq, ids, log_weights, samples,
                                               static_cast<const abx::bf16*>(text_k),
                                               static_cast<const abx::bf16*>(text_v), text_tokens,
                                               static_cast<abx::bf16*>(o), lse, workspace, workspace_bytes, stream),
                      "paired prefill launch");
}

int abx_dense_prefill(const void* q, const void* k, const void* v, int64_t bh, int64_t seq, void* o, float* lse,
                      abx_stream_t stream) {
    if (int st = check_qk_shape(bh, seq)) return st;
    if (!q || !k || !v || !o) return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, v and o must be non-null");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q, k, v and o must be 16-byte aligned");
    return check_cuda(abx::launch_prefill(static_cast<const abx::bf16*>(q), seq, static_cast<const abx::bf16*>(k),
                                          static_cast<const abx::bf16*>(v), bh, seq, nullptr, nullptr,
                                          seq / abx::kKv4, nullptr, nullptr, 0, static_cast<abx::bf16*>(o), lse,
                                          stream),
                      "prefill launch");
}

int abx_cross_prefill(const void* q, int64_t q_tokens, const void* k, const void* v, int64_t kv_tokens, int64_t bh,
                      const int32_t* ids, const float* log_weights, int64_t samples, const void* text_k,
                      const void* text_v, int64_t text_tokens, void* o, float* lse, abx_stream_t stream) {
    if (bh <= 0 || q_tokens <= 0) return fail(ABX_ERR_INVALID_ARGUMENT, "bad query shape");
    if (kv_tokens < 0 || kv_tokens % abx::kKv4 != 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "key token count must be a non-negative multiple of 4");
    if (kv_tokens / abx::kKv4 > abx::kMaxFineBlocks)
        return fail(ABX_ERR_UNSUPPORTED, "more than %d key blocks", abx::kMaxFineBlocks);
    if (!q || !o || !aligned16(q) || !aligned16(o))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q and o must be non-null and 16-byte aligned");
    if (samples < 0 || samples > kv_tokens / abx::kKv4)
        return fail(ABX_ERR_INVALID_ARGUMENT, "samples must be in [0, kv_tokens/4] (got %lld)", (long long)samples);
    if (samples > 0 && (!k || !v || !aligned16(k) || !aligned16(v)))
        return fail(ABX_ERR_INVALID_ARGUMENT, "k and v must be non-null and 16-byte aligned");
    if ((ids == nullptr) != (log_weights == nullptr))
        return fail(ABX_ERR_INVALID_ARGUMENT, "ids and log_weights are given together (or neither: dense)");
    if (text_tokens < 0) return fail(ABX_ERR_INVALID_ARGUMENT, "negative text token count");
    if (text_tokens > 0 && (!text_k || !text_v || !aligned16(text_k) || !aligned16(text_v)))
        return fail(ABX_ERR_INVALID_ARGUMENT, "text_k/text_v must be non-null and 16-byte aligned");
    if (samples + (text_tokens + abx::kKv4 - 1) / abx::kKv4 <= 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "every row needs at least one key");
    return check_cuda(abx::launch_prefill(static_cast<const abx::bf16*>(q), q_tokens,
                                          static_cast<const abx::bf16*>(k), static_cast<const abx::bf16*>(v), bh,
                                          kv_tokens, ids, log_weights, samples,
                                          static_cast<const abx::bf16*>(text_k),
                                          static_cast<const abx::bf16*>(text_v), text_tokens,
                                          static_cast<abx::bf16*>(o), lse, stream),
                      "prefill launch");
}

int abx_selftest_wait_timeout(int64_t limit_cycles, abx_stream_t stream) {
    if (limit_cycles <= 0 || limit_cycles > 4000000000LL)
        return fail(ABX_ERR_INVALID_ARGUMENT, "limit must be in (0, 4e9] cycles");
    abx::wait_selftest_kernel<<<1, 64, 0, stream>>>(static_cast<uint64_t>(limit_cycles), abx::device_error_word());
    return check_cuda(cudaGetLastError(), "self-test launch");
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Streaming operators: rotary positions, cache append, chunk attention.
// ---------------------------------------------------------------------------
namespace {

// Every row (batch, head, token) of a [.., 128] tensor starts on a 16-byte boundary.
int check_rows(const char* name, const void* p, const int64_t (&stride)[3], int element_bytes) {
    if (p == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "%s must be non-null", name);
    if (!aligned16(p)) return fail(ABX_ERR_INVALID_ARGUMENT, "%s must be 16-byte aligned", name);
    for (int64_t s : stride)
        if (s < 0 || s * element_bytes % 16 != 0)
            return fail(ABX_ERR_INVALID_ARGUMENT, "the strides of %s must be multiples of 16 bytes (got %lld elements)",
                        name, (long long)s);
    return ABX_OK;
}

int check_pages(int64_t sequences, int64_t table_width, int64_t page_size, int64_t pages) {
    if (sequences < 1 || sequences > 0x3fffffff) return fail(ABX_ERR_INVALID_ARGUMENT, "there must be at least one sequence");
    if (page_size < 16 || (page_size < 128 ? (page_size & (page_size - 1)) != 0 : page_size % 128 != 0))
        return fail(ABX_ERR_INVALID_ARGUMENT, "page size must be 16, 32, 64 or a multiple of 128 (got %lld)", (long long)page_size);
    if (pages < 1 || pages > 0x3fffffff) return fail(ABX_ERR_INVALID_ARGUMENT, "the cache must have pages (got %lld)", (long long)pages);
    if (table_width < 1) return fail(ABX_ERR_INVALID_ARGUMENT, "the page table must have columns");
    if (page_size > abx::kMaxCacheKeys || table_width > abx::kMaxCacheKeys / page_size)
        return fail(ABX_ERR_UNSUPPORTED, "more than 2^30 cache positions a sequence");
    return ABX_OK;
}

// Whether a dim of more than one element repeats its rows by a stride of 0.
bool repeats(const int64_t (&size)[3], const int64_t (&stride)[3]) {
    for (int i = 0; i < 3; ++i)
        if (size[i] > 1 && stride[i] == 0) return true;
    return false;
}

// Four dims [128, d1, d2, d3] with strides in elements and 64 x b1 x b2 x 1 boxes, 128-byte swizzle. A
// dim of one element may have any stride; the map wants one that it can encode. Rows that repeat are refused: the
// encoder takes a stride of 0, but nothing documents what a copy then does.
cudaError_t encode_rows4d(CUtensorMap* map, const void* base, bool fp16, const int64_t (&size)[3], const int64_t (&stride)[3],
                          uint32_t b1, uint32_t b2) {
    auto encode = abx::tensor_map_encoder();
    if (encode == nullptr) return cudaErrorNotSupported;
    if (repeats(size, stride)) return cudaErrorInvalidValue;
    cuuint64_t dims[4] = {abx::kHeadDim}, bytes[3];
    for (int i = 0; i < 3; ++i) {
        dims[i + 1] = static_cast<cuuint64_t>(size[i]);
        bytes[i] = static_cast<cuuint64_t>(size[i] > 1 ? stride[i] : abx::kHeadDim) * 2;
    }
    const cuuint32_t box[4] = {64, b1, b2, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// K or V: [128, tokens of a page, kv_heads, pages] from strides (page, head, token).
cudaError_t encode_cache(CUtensorMap* map, const void* base, bool fp16, int64_t tokens, int64_t heads, int64_t pages,
                         const int64_t (&stride)[3], uint32_t box_rows) {
    const int64_t size[3] = {tokens, heads, pages}, steps[3] = {stride[2], stride[1], stride[0]};
    return encode_rows4d(map, base, fp16, size, steps, box_rows, 1);
}

int64_t at_most(int64_t x, int64_t most) { return x < most ? x : most; }

// Checks every argument of a chunk call that does not need the device, and lays the call out.
int chunk_plan(const abx_chunk_args* c, abx::ChunkArgs& a, size_t& workspace) {
    if (c == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "args is null");
    if (c->dtype != ABX_BF16 && c->dtype != ABX_FP16) return fail(ABX_ERR_INVALID_ARGUMENT, "attention takes bf16 or fp16");
    const bool paged = c->page_table != nullptr;
    if (c->sequences < 1 || c->tokens < 1) return fail(ABX_ERR_INVALID_ARGUMENT, "there must be sequences and tokens");
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->heads < 1 || c->heads % c->kv_heads != 0)
        return fail(ABX_ERR_INVALID_ARGUMENT, "heads (%lld) must be a multiple of kv_heads (%lld)", (long long)c->heads,
                    (long long)c->kv_heads);
    if (c->window < 0 || c->sinks < 0 || c->block < 1)
        return fail(ABX_ERR_INVALID_ARGUMENT, "window and sinks must not be negative, block must be positive");
    if (int st = check_rows("q", c->q, c->q_stride, 2)) return st;
    if (int st = check_rows("k", c->k, c->k_stride, 2)) return st;
    if (int st = check_rows("v", c->v, c->v_stride, 2)) return st;
    if (int st = check_rows("o", c->o, c->o_stride, 2)) return st;
    if (c->longest < 1 || c->longest > c->tokens)
        return fail(ABX_ERR_INVALID_ARGUMENT, "longest must be in [1, tokens] (got %lld)", (long long)c->longest);
    if (paged) {
        if (int st = check_pages(c->sequences, c->table_width, c->page_size, c->pages)) return st;
        if (c->starts == nullptr || c->lengths == nullptr)
            return fail(ABX_ERR_INVALID_ARGUMENT, "starts and lengths must be non-null");
    } else {
        if (c->keys < 1) return fail(ABX_ERR_INVALID_ARGUMENT, "there must be keys");
        if (c->keys > abx::kMaxCacheKeys || c->sequences > 0x3fffffff) return fail(ABX_ERR_UNSUPPORTED, "more than 2^30 keys");
        if (c->longest != c->tokens) return fail(ABX_ERR_INVALID_ARGUMENT, "longest must be the token count");
    }
    const int64_t cache[3] = {paged ? c->pages : c->sequences, c->kv_heads, paged ? c->page_size : c->keys};
    if (repeats(cache, c->k_stride) || repeats(cache, c->v_stride))
        return fail(ABX_ERR_INVALID_ARGUMENT, "the rows of k and v must not repeat by a stride of 0");
    const int64_t all_tokens = paged ? c->tokens : c->tokens * c->sequences;
    if (c->heads > 0x3fffffff || c->tokens > 0x3fffffff / c->heads || all_tokens > 0x7fffffff)
        return fail(ABX_ERR_UNSUPPORTED, "too many query rows");
    // Positions stay below 2^30, so a block that is larger is one block over all of them; its window counts back
    // from the block's end, and what of it lies past the largest block here hides no key.
    const int64_t largest = 0x3fffffff, past = c->block > largest ? c->block - largest : 0;
    const int64_t window = c->window > past ? c->window - past : 0;
    a = abx::ChunkArgs{};
    a.q = c->q;
    a.o = c->o;
    a.lse = c->lse;
    a.q_seq = paged ? 0 : c->q_stride[0], a.q_head = c->q_stride[1], a.q_token = c->q_stride[2];
    a.o_seq = paged ? 0 : c->o_stride[0], a.o_head = c->o_stride[1], a.o_token = c->o_stride[2];
    a.l_seq = paged ? 0 : c->lse_stride[0], a.l_head = c->lse_stride[1], a.l_token = c->lse_stride[2];
    a.starts = paged ? c->starts : nullptr;
    a.lengths = paged ? c->lengths : nullptr;
    a.table = c->page_table;
    a.seqs = static_cast<int32_t>(c->sequences);
    a.heads = static_cast<int32_t>(c->heads);
    a.kv_heads = static_cast<int32_t>(c->kv_heads);
    a.group = static_cast<int32_t>(c->heads / c->kv_heads);
    a.tokens = static_cast<int32_t>(c->tokens);
    a.longest = static_cast<int32_t>(c->longest);
    a.keys = static_cast<int32_t>(paged ? c->table_width * c->page_size : c->keys);
    a.table_width = static_cast<int32_t>(paged ? c->table_width : 0);
    a.page_size = static_cast<int32_t>(paged ? c->page_size : 0);
    a.page_shift = -1;
    for (int shift = 4; shift < 30; ++shift)
        if (a.page_size == 1 << shift) a.page_shift = shift;
    a.pages = static_cast<int32_t>(paged ? c->pages : c->sequences);
    a.window = c->window == 0 ? abx::kNoWindow : static_cast<int32_t>(at_most(window, abx::kNoWindow - 1));
    a.sinks = c->window == 0 ? 0 : static_cast<int32_t>(at_most(c->sinks, largest));
    a.block = static_cast<int32_t>(at_most(c->block, largest));
    a.rows_total = all_tokens * c->heads;
    a.kappa = abx::qk_scale_log2();
    abx::chunk_layout(a);
    workspace = a.splits > 1 && !a.cluster ? align_up(static_cast<size_t>(a.splits) * a.rows_total * abx::kHeadDim * 4) +
                                   align_up(static_cast<size_t>(a.splits) * a.rows_total * 4)
                             : 0;
    return ABX_OK;
}

}  // namespace

extern "C" {

int abx_rotary(const abx_rotary_args* r, abx_stream_t stream) {
    if (r == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "args is null");
    const bool paged = r->page_table != nullptr;
    if (r->dtype != ABX_BF16 && r->dtype != ABX_FP16 && (paged || r->dtype != ABX_F32))
        return fail(ABX_ERR_INVALID_ARGUMENT, "rotary takes bf16, fp16 or (without a cache) f32");
    const int e = r->dtype == ABX_F32 ? 4 : 2;
    if (r->batch < 1 || r->tokens < 1 || (paged && r->batch != 1))
        return fail(ABX_ERR_INVALID_ARGUMENT, "there must be tokens (one batch of them with a page table)");
    if (r->tokens > 0x7fffffff / r->batch) return fail(ABX_ERR_UNSUPPORTED, "too many tokens");
    if (r->heads < 0 || r->kv_heads < 0 || r->heads > 0xffffff || r->kv_heads > 0xffffff)
        return fail(ABX_ERR_INVALID_ARGUMENT, "bad head count");
    const bool has_q = r->q != nullptr, has_k = r->k != nullptr;
    if ((!has_q && !has_k) || (has_q && r->heads < 1) || (has_k && r->kv_heads < 1) || (paged && !has_k))
        return fail(ABX_ERR_INVALID_ARGUMENT, "q or k (with a page table, k and v) must be given with their heads");
    if (has_q || !paged) {
        if (r->positions == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "positions must be non-null");
    }
    abx::RotaryArgs a{};
    if (r->positions != nullptr) {
        if (r->axes < 1 || r->axes > abx::kRotaryAxes)
            return fail(ABX_ERR_INVALID_ARGUMENT, "between 1 and %d axes (got %d)", abx::kRotaryAxes, r->axes);
        if (!(r->theta > 0) || !std::isfinite(r->theta)) return fail(ABX_ERR_INVALID_ARGUMENT, "theta must be positive");
        int dims = 0;
        for (int x = 0; x < r->axes; ++x) {
            if (r->sections[x] < 0 || r->sections[x] > abx::kHeadDim || r->sections[x] % 2 != 0)
                return fail(ABX_ERR_INVALID_ARGUMENT, "sections must be even");
            dims += r->sections[x];
        }
        if (dims != abx::kHeadDim) return fail(ABX_ERR_INVALID_ARGUMENT, "sections must sum to 128 (got %d)", dims);
        // The frequencies follow from the axes alone: worked out when those change (0.7 us of a call's host time).
        struct Table {
            int32_t axes, sections[abx::kRotaryAxes], shared;
            double theta;
            double freq[abx::kPairs];
            uint8_t axis[abx::kPairs];
        };
        thread_local Table table{};
        if (table.axes != r->axes || table.shared != (r->shared != 0) || table.theta != r->theta ||
            std::memcmp(table.sections, r->sections, sizeof(int32_t) * r->axes) != 0) {
            const double log_theta = std::log(r->theta);
            int pair = 0;
            for (int x = 0; x < r->axes; ++x)
                for (int i = 0; i < r->sections[x] / 2; ++i, ++pair) {
                    const double power = r->shared ? 2.0 * pair / abx::kHeadDim : 2.0 * i / r->sections[x];
                    table.freq[pair] = std::exp(-power * log_theta) / 3.14159265358979323846;
                    table.axis[pair] = static_cast<uint8_t>(x);
                }
            table.axes = r->axes;
            table.shared = r->shared != 0;
            table.theta = r->theta;
            std::memcpy(table.sections, r->sections, sizeof(int32_t) * r->axes);
        }
        std::memcpy(a.freq, table.freq, sizeof(a.freq));
        std::memcpy(a.axis, table.axis, sizeof(a.axis));
    }
    auto add = [&](const char* name, const void* src, const int64_t (&s)[3], void* dst, const int64_t (&d)[3],
                   int64_t heads, bool turn, bool to_cache) -> int {
        if (int st = check_rows(name, src, s, e)) return st;
        if (int st = check_rows("the output", dst, d, e)) return st;
        abx::RotaryJob& j = a.job[a.jobs++];
        j = abx::RotaryJob{src, dst, s[0], s[1], s[2], d[0], d[1], d[2], static_cast<int32_t>(heads), turn, to_cache};
        a.heads += j.heads;
        return ABX_OK;
    };
    if (has_q)
        if (int st = add("q", r->q, r->q_stride, r->q_out, r->q_out_stride, r->heads, true, false)) return st;
    if (has_k)
        if (int st = add("k", r->k, r->k_stride, r->k_out, r->k_out_stride, r->kv_heads, r->positions != nullptr, paged))
            return st;
    if (paged) {
        if (int st = add("v", r->v, r->v_stride, r->v_out, r->v_out_stride, r->kv_heads, false, true)) return st;
        if (int st = check_pages(r->sequences, r->table_width, r->page_size, r->pages)) return st;
        if (r->starts == nullptr || r->lengths == nullptr)
            return fail(ABX_ERR_INVALID_ARGUMENT, "starts and lengths must be non-null");
        a.starts = r->starts;
        a.lengths = r->lengths;
        a.table = r->page_table;
        a.seqs = static_cast<int32_t>(r->sequences);
        a.table_width = static_cast<int32_t>(r->table_width);
        a.page_size = static_cast<int32_t>(r->page_size);
        a.pages = static_cast<int32_t>(r->pages);
    }
    a.positions = r->positions;
    a.p_batch = r->positions_batch;
    a.axes = r->axes;
    a.batch = static_cast<int32_t>(r->batch);
    a.tokens = static_cast<int32_t>(r->tokens);
    a.halves = r->halves != 0;
    a.sign = r->inverse ? -1.f : 1.f;
    a.error = abx::device_error_word();
    return check_cuda(abx::launch_rotary(a, r->dtype, stream), "rotary launch");
}

int abx_chunk_workspace_size(const abx_chunk_args* args, size_t* bytes) {
    if (bytes == nullptr) return fail(ABX_ERR_INVALID_ARGUMENT, "bytes is null");
    abx::ChunkArgs a;
    return chunk_plan(args, a, *bytes);
}

int abx_chunk_attention(const abx_chunk_args* args, void* workspace, size_t workspace_bytes, abx_stream_t stream) {
    abx::ChunkArgs a;
    size_t need = 0;
    if (int st = chunk_plan(args, a, need)) return st;
    if (need > 0) {
        if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % kAlign != 0)
            return fail(ABX_ERR_WORKSPACE, "workspace must be non-null and 256-byte aligned");
        if (workspace_bytes < need)
            return fail(ABX_ERR_WORKSPACE, "workspace too small (%zu < %zu bytes)", workspace_bytes, need);
        a.part_o = static_cast<float*>(workspace);
        a.part_lse = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                              align_up(static_cast<size_t>(a.splits) * a.rows_total * abx::kHeadDim * 4));
    }
    a.error = abx::device_error_word();
    const bool fp16 = args->dtype == ABX_FP16;
    const int box_rows = a.table == nullptr || a.page_size > abx::kChunkBoxKeys ? abx::kChunkBoxKeys : a.page_size;
    const int64_t tokens = a.table == nullptr ? a.keys : a.page_size;
    abx::ChunkMaps maps{};
    if (int st = check_cuda(encode_cache(&maps.k, args->k, fp16, tokens, a.kv_heads, a.pages, args->k_stride, box_rows),
                            "tensor map of k"))
        return st;
    if (int st = check_cuda(encode_cache(&maps.v, args->v, fp16, tokens, a.kv_heads, a.pages, args->v_stride, box_rows),
                            "tensor map of v"))
        return st;
    if (a.tile_rows == 256 && 128 % a.group == 0) {
        // Queries by TMA where a box holds 128 rows in order; rows that repeat (a stride of 0) or that no map
        // can describe are loaded one by one.
        const int64_t size[3] = {a.heads, a.tokens, a.table == nullptr ? a.seqs : 1};
        const int64_t steps[3] = {a.q_head, a.q_token, a.q_seq};
        a.q_map = encode_rows4d(&maps.q, args->q, fp16, size, steps, a.group, 128 / a.group) == cudaSuccess;
    }
    if (int st = check_cuda(abx::launch_chunk(a, maps, fp16, box_rows, stream), "chunk attention launch")) return st;
    return need > 0 ? check_cuda(abx::launch_chunk_join(a, fp16, stream), "chunk join launch") : ABX_OK;
}

}  // extern "C"
