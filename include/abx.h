/*
 * abx.h — C ABI of the B200 (sm_100a) AB-Attention sparse-attention hot path.
 *
 * The reference binds its kernels through a pybind11 module (`ab_attention._C`,
 * csrc/bindings.cpp:3-8, csrc/ops.h:5-8) and runs the sparse prefill through
 * FlashInfer (ab_attention/flashinfer_backend.py:164-242). This header is the
 * replacement boundary: plain pointers, sizes and a cudaStream_t, no torch types.
 *
 * Conventions shared by every entry point:
 *   - Tensors are dense, row-major, on the current CUDA device. `bh` is batch*heads,
 *     `seq` the token count; q/k/v are bf16 [bh, seq, 128] (head dim fixed at 128
 *     as in csrc/ibcs.cu:32 and flashinfer_backend.py:19).
 *   - qb = ceil(seq/128) query blocks, F = seq/4 KV4 blocks, rows = bh*qb.
 *   - Every call is asynchronous on `stream` and returns an abx_status; 0 is success.
 *     The caller owns every buffer, including workspaces sized by *_workspace_size.
 *   - bf16 / fp16 buffers are passed as `void*` / `uint16_t*` (raw 16-bit words).
 */
#ifndef ABX_H_
#define ABX_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct CUstream_st* abx_stream_t; /* identical to cudaStream_t */

enum abx_status {
  ABX_OK = 0,
  ABX_ERR_INVALID_ARGUMENT = 1, /* null pointer, bad shape or size                      */
  ABX_ERR_UNSUPPORTED = 2,      /* shape outside a kernel limit (F > 32768, smem cap)  */
  ABX_ERR_WORKSPACE = 3,        /* workspace missing, too small or misaligned           */
  ABX_ERR_CUDA = 4,             /* a CUDA runtime call or kernel launch failed          */
  ABX_ERR_DEVICE_TIMEOUT = 5    /* a bounded device-side wait gave up (see abx_device_status) */
};

/* Library identification and error text. abx_last_error() is thread-local. */
int abx_version(void);
const char* abx_status_string(int status);
const char* abx_last_error(void);

/* Sticky device-side error word for the current device (0 = none): set by a
 * kernel whose bounded wait expired. Reading it synchronizes `stream`; pass
 * clear=1 to reset it. */
int abx_device_status(abx_stream_t stream, int clear, int* status_out);

/* Self-test of the device-side failure path (no counterpart in the reference):
 * two warps wait, bounded by limit_cycles SM clock cycles, on an mbarrier that
 * nothing arrives at, one with the polling and one with the suspending form of
 * the library's bounded wait; both give up, the kernel returns normally and the
 * device error word reads ABX_ERR_DEVICE_TIMEOUT. The context stays usable. */
int abx_selftest_wait_timeout(int64_t limit_cycles, abx_stream_t stream);

/* ---------------------------------------------------------------------------
 * IBCS stages (parity entry points). Each mirrors one reference kernel.
 * ------------------------------------------------------------------------- */

/* cluster_queries_kernel (csrc/ibcs.cu:106-238): farthest-first 8-way clustering
 * of each 128-query block. Outputs (any may be NULL except populations):
 *   centroids        bf16 [rows, 8, 128]   bf16_rn(mean of members), 0 if empty
 *   scaled_centroids bf16 [rows, 8, 128]   bf16_rn(centroid * 128^-0.5 * log2 e)
 *                                          (the MMA operand, csrc/ibcs.cu:293-295)
 *   populations      f32  [rows, 8]        member counts (the reference stores fp16)
 *   assignments      i32  [rows, 128]      centroid slot per query, -1 past the end */
int abx_ibcs_cluster(const void* q, int64_t bh, int64_t seq, void* centroids,
                     void* scaled_centroids, float* populations, int32_t* assignments,
                     abx_stream_t stream);

/* pool_keys_kernel (csrc/ibcs.cu:244-266): two representatives per KV4 block,
 * bf16_rn(0.5*(k[4j+2t] + k[4j+2t+1])). pooled: bf16 [bh, F, 2, 128]. */
int abx_ibcs_pool(const void* k, int64_t bh, int64_t seq, void* pooled, abx_stream_t stream);

/* ibcs_lse_kernel (csrc/ibcs.cu:370-489): per (row, centroid, KV4 block) the fp16
 * pair log2-sum-exp of the two scaled centroid.key scores, plus each (row,
 * centroid)'s running normalizer. lse: fp16 [rows, 8, F]; lse_max/lse_den: f32 [rows, 8]. */
int abx_ibcs_lse(const void* scaled_centroids, const void* pooled, int64_t bh, int64_t qb,
                 int64_t fine_blocks, uint16_t* lse, float* lse_max, float* lse_den,
                 abx_stream_t stream);

/* ibcs_scores_kernel (csrc/ibcs.cu:495-538): population-weighted mixture of the
 * eight centroid distributions. scores: f32 [rows, F]. */
int abx_ibcs_mix(const uint16_t* lse, const float* populations, const float* lse_max,
                 const float* lse_den, int64_t rows, int64_t fine_blocks, float* scores,
                 abx_stream_t stream);

/* ---------------------------------------------------------------------------
 * Replacements for the reference native ops.
 * ------------------------------------------------------------------------- */

/* Workspace for abx_ibcs_scores and abx_build_plan (bytes, 256-byte aligned base). */
int abx_ibcs_workspace_size(int64_t bh, int64_t seq, size_t* bytes);

/* `_C.ibcs(q, k) -> scores` (csrc/ibcs.cu:549-617): all four IBCS stages.
 * scores: f32 [rows, F]. */
int abx_ibcs_scores(const void* q, const void* k, int64_t bh, int64_t seq, float* scores,
                    void* workspace, size_t workspace_bytes, abx_stream_t stream);

/* `_C.sip(scores, offsets, ids, logs)` (csrc/sip.cu:170-199): iterative pi=1
 * certainty then systematic sampling without replacement. scores f32 [rows,
 * population], offsets f32 [rows] in [0,1), ids i32 [rows, samples] and
 * log_weights f32 [rows, samples] written in place. 0 < samples < population. */
int abx_sip(const float* scores, const float* offsets, int64_t rows, int64_t population,
            int32_t* ids, float* log_weights, int64_t samples, abx_stream_t stream);

/* build_plan's device work (ab_attention/attention.py:27-82) in one call:
 * IBCS with the mixture fused into SIP, so the per-block scores never reach HBM.
 * ids/log_weights: [rows, samples]. Same results as abx_ibcs_scores + abx_sip. */
int abx_build_plan(const void* q, const void* k, int64_t bh, int64_t seq,
                   const float* offsets, int64_t samples, int32_t* ids, float* log_weights,
                   void* workspace, size_t workspace_bytes, abx_stream_t stream);

/* abx_build_plan without a workspace argument, for callers that cannot call
 * cudaMalloc (device memory owned by another allocator or reserved up front, or
 * a path where cudaMalloc's implicit synchronisation is not acceptable). No
 * counterpart in the reference. It allocates nothing: its scratch is a fixed
 * file-scope device array of abx_static_scratch_bytes() (256 MiB) that every GPU
 * loading libabx holds until exit, so one head of the input must fit in it
 * (about 90k tokens); larger inputs are rejected with ABX_ERR_WORKSPACE. Heads
 * are processed in passes that fit the array. The first call on a device looks
 * up the array's device address (make it before any stream capture). All calls
 * share the array: calls that overlap on the GPU (different streams, or
 * different host threads) race, so serialise them. Results equal abx_build_plan's. */
size_t abx_static_scratch_bytes(void);
int abx_build_plan_static(const void* q, const void* k, int64_t bh, int64_t seq,
                          const float* offsets, int64_t samples, int32_t* ids,
                          float* log_weights, abx_stream_t stream);

/* ---------------------------------------------------------------------------
 * Sparse prefill: replaces flashinfer_backend.paged_attention
 * (ab_attention/flashinfer_backend.py:164-242) and its ABSipAttention variant (:30-58).
 * For each row (bh, query block) the keys are the KV4 blocks ids[row, 0..samples)
 * (local to the head), each with logit shift log_weights[row, slot] in log2 units,
 * followed by `text_tokens` always-included keys from text_k/text_v
 * ([bh, text_tokens, 128], shift 0; NULL when text_tokens == 0).
 *   o   bf16 [bh, seq, 128]
 *   lse f32  [bh, seq] base-2 log-sum-exp of the scaled logits (NULL to skip)
 * ------------------------------------------------------------------------- */
int abx_sparse_prefill(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                       const int32_t* ids, const float* log_weights, int64_t samples,
                       const void* text_k, const void* text_v, int64_t text_tokens,
                       void* o, float* lse, abx_stream_t stream);

/* abx_sparse_prefill with two adjacent query blocks of a head per CTA, fed from
 * one gather of the union of their samples (same results up to the order of
 * the floating-point sums). `workspace` (device memory, any alignment) holds the
 * per-pair union lists; abx_prefill_workspace_size() gives its size, 0 when the
 * shape cannot be paired (more than 65,534 slots, or a map of seq/4 slots
 * larger than shared memory), in which case this call is abx_sparse_prefill and
 * ignores the workspace. Same replaced interface as abx_sparse_prefill. */
int abx_prefill_workspace_size(int64_t bh, int64_t seq, int64_t samples, int64_t text_tokens, size_t* bytes);
int abx_sparse_prefill_paired(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                              const int32_t* ids, const float* log_weights, int64_t samples,
                              const void* text_k, const void* text_v, int64_t text_tokens,
                              void* o, float* lse, void* workspace, size_t workspace_bytes,
                              abx_stream_t stream);

/* The two launches of abx_sparse_prefill_paired as separate calls (no
 * counterpart in the reference). abx_pair_plan writes each pair's union list
 * for `ids` into the workspace; abx_sparse_prefill_paired_planned runs the
 * prefill from those lists, which must have been written by abx_pair_plan for
 * the same ids, shape and text count (the kernel range-checks every list entry,
 * so stale lists give wrong results and ABX_ERR_INVALID_ARGUMENT, never an
 * out-of-bounds read). A plan reused over several calls (the video schedule
 * keeps a plan for four denoising steps) builds its lists once. Both return
 * ABX_ERR_UNSUPPORTED for a shape abx_prefill_workspace_size reports as 0. */
int abx_pair_plan(const int32_t* ids, int64_t bh, int64_t seq, int64_t samples, int64_t text_tokens,
                  void* workspace, size_t workspace_bytes, abx_stream_t stream);
int abx_sparse_prefill_paired_planned(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                                      const int32_t* ids, const float* log_weights, int64_t samples,
                                      const void* text_k, const void* text_v, int64_t text_tokens, void* o,
                                      float* lse, void* workspace, size_t workspace_bytes, abx_stream_t stream);

/* CUDA IPC of an output buffer between the processes of one node (no
 * counterpart in the reference): abx_ipc_handle gives the 64-byte handle of the
 * allocation holding `ptr` and ptr's byte offset in it; another process opens
 * it with abx_ipc_open (the mapping is made for the caller's current device,
 * with peer access enabled to the owner's device) and adds the offset, then
 * closes it with abx_ipc_close. */
int abx_ipc_handle(const void* ptr, void* handle, size_t* offset);
int abx_ipc_open(const void* handle, void** base);
int abx_ipc_close(void* base);

/* Asynchronous copy of `bytes` on `stream`, either address possibly another
 * GPU's (a mapping opened by abx_ipc_open): between GPUs it runs on a copy
 * engine over NVLink and uses no SMs. No counterpart in the reference. */
int abx_peer_copy(void* dst, const void* src, size_t bytes, abx_stream_t stream);

/* The paired prefill (pair plan included) with its output rows written straight
 * into `num_outs` (1..8) copies of the whole layer's output, each [out_heads,
 * seq, 128] bf16, at heads [out_head_base, out_head_base + bh): on several GPUs,
 * one copy per rank, the other ranks' reached through their mapped (CUDA IPC)
 * addresses, so a head-sharded layer needs no all-gather afterwards. No
 * counterpart in the reference (it has no multi-GPU path); it replaces the NCCL
 * all-gather of the sharded outputs. The stores are plain peer stores over
 * NVLink, made visible system-wide before the kernel ends; the caller orders a
 * reader on another GPU after this call with any collective (an all-reduce of
 * one element) issued on `stream` after it. lse (optional) is this call's heads
 * only, [bh, seq]. ABX_ERR_UNSUPPORTED for a shape that cannot be paired. */
int abx_sparse_prefill_scatter(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                               const int32_t* ids, const float* log_weights, int64_t samples,
                               const void* text_k, const void* text_v, int64_t text_tokens,
                               void* const* outs, int num_outs, int64_t out_head_base, int64_t out_heads,
                               float* lse, void* workspace, size_t workspace_bytes, abx_stream_t stream);

/* Dense attention through the same prefill kernel (every KV4 block, shift 0):
 * the dense comparator. o / lse as above. */
int abx_dense_prefill(const void* q, const void* k, const void* v, int64_t bh, int64_t seq,
                      void* o, float* lse, abx_stream_t stream);

/* Queries attending to keys of another length: q [bh, q_tokens, 128] against
 * the KV4 granules named by ids ([bh * ceil(q_tokens/128), samples]; NULL ids
 * and log_weights = the first `samples` granules of k/v in order, weight 0)
 * of k, v [bh, kv_tokens, 128], followed by the text keys text_k, text_v
 * [bh, text_tokens, 128] (any count; keys past text_tokens in the last
 * granule are masked). o [bh, q_tokens, 128], lse [bh, q_tokens] (base 2) or
 * NULL. No counterpart entry point in the reference: it covers the
 * HunyuanVideo partitions its video.py:129-151 runs through FlashInfer (text
 * queries over all video + text keys, and the padding partition with
 * samples = 0 and the padding tokens as text keys). */
int abx_cross_prefill(const void* q, int64_t q_tokens, const void* k, const void* v, int64_t kv_tokens, int64_t bh,
                      const int32_t* ids, const float* log_weights, int64_t samples, const void* text_k,
                      const void* text_v, int64_t text_tokens, void* o, float* lse, abx_stream_t stream);

/* ---------------------------------------------------------------------------
 * Streaming operators (no counterpart in the reference): rotary positions, a paged
 * key/value cache, and attention of new tokens over it. Element types: bf16 or
 * fp16 (rotary without a cache also f32); head dim 128. Strides are in elements,
 * the innermost dim is contiguous, and every row starts on a 16-byte boundary.
 * ------------------------------------------------------------------------- */
enum abx_dtype { ABX_BF16 = 0, ABX_FP16 = 1, ABX_F32 = 2 };

/* Rotary positions over up to four axes. Axis a turns sections[a] of the head's
 * 128 dims (even; they sum to 128), in order. Pair i of an axis with d dims turns
 * by position * theta^(-2i / d), or, shared, pair i of the whole head (of its 64)
 * by position * theta^(-2i / 128). Pairs are dims (2i, 2i + 1), or, halves,
 * (i, i + 64). inverse turns back, which is also the turn's gradient. Angles are
 * taken in 64 bits.
 *
 * q, k, v are rows (batch, head, token); q_out and k_out get the turned rows. Any
 * of the three may be NULL (with its heads 0). positions: int32 [batch or 1,
 * tokens, axes]. v is only used with a page table.
 *
 * With page_table the call appends to a cache: batch is 1, tokens are packed
 * (sequence s owns tokens [starts[s], starts[s + 1]), and its last token goes to
 * cache position lengths[s] - 1), and k_out / v_out are the cache, strides (page,
 * head, token of a page), both [pages, kv_heads, page_size, 128]. positions may be
 * NULL: k is stored as it is (and q must be NULL). A token outside every
 * sequence is not stored; one whose place is outside the table, or whose table
 * entry names no page, is not stored and records ABX_ERR_INVALID_ARGUMENT in the
 * device error word. Two tokens with one place leave parts of either's row. */
typedef struct abx_rotary_args {
  int32_t dtype;
  int32_t axes;
  int32_t sections[4];
  double theta;
  int32_t shared, halves, inverse;
  const int32_t* positions;
  int64_t positions_batch; /* stride of positions between batches, 0: one for all */
  int64_t batch, tokens;
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;
  int64_t heads, kv_heads;
  int64_t q_stride[3], k_stride[3], v_stride[3]; /* batch, head, token */
  int64_t q_out_stride[3], k_out_stride[3], v_out_stride[3];
  const int32_t *starts, *lengths, *page_table; /* [sequences + 1], [sequences], [sequences, table_width] */
  int64_t sequences, table_width, page_size, pages;
} abx_rotary_args;
int abx_rotary(const abx_rotary_args* args, abx_stream_t stream);

/* Attention (scale 128^-0.5) of new tokens over the keys so far, those of the new
 * tokens included. Token i of a sequence with n new tokens and `len` keys is at
 * position p = len - n + i and sees key j when j < min(e, len) and (j >= e - window
 * or j < sinks), e = (p / block + 1) * block, none for p < 0: causal for block 1; a
 * block of tokens otherwise sees to its own end. window 0: no limit. A row that
 * sees nothing gives zeros and an lse of -inf. heads is a multiple of kv_heads; head
 * h reads key head h / (heads / kv_heads).
 *
 * Contiguous (page_table NULL): q and o rows (sequence, head, token) of `tokens`
 * tokens a sequence, k and v rows (sequence, head, token) of `keys` tokens. Rows of
 * q may repeat (a stride of 0), those of k and v may not.
 * Paged: tokens are packed (`tokens` of all sequences; starts / lengths as above; the
 * sequence strides of q, o and lse are ignored), k and v are rows (page, head, token
 * of a page). page_size is 16, 32, 64 or a multiple of 128. longest bounds the tokens
 * of any sequence; a sequence with more is not computed (its rows are left as they
 * were) and records ABX_ERR_INVALID_ARGUMENT, as do lengths or starts past the buffers (clipped)
 * and table entries that name no page (read as zeros). Rows of tokens in no
 * sequence are left as they were. The cached rows of a sequence have to be
 * finite; what lies behind them in its last page may be anything.
 *   lse f32 rows (sequence, head, token), base 2; NULL to skip.
 * The workspace (device memory, 256-byte aligned) joins keys that several CTAs
 * share; abx_chunk_workspace_size may report 0. */
typedef struct abx_chunk_args {
  int32_t dtype;
  const void *q, *k, *v;
  void* o;
  float* lse;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3], lse_stride[3];
  int64_t sequences, tokens, longest, keys, heads, kv_heads;
  const int32_t *starts, *lengths, *page_table;
  int64_t table_width, page_size, pages;
  int64_t window, sinks, block;
} abx_chunk_args;
int abx_chunk_workspace_size(const abx_chunk_args* args, size_t* bytes);
int abx_chunk_attention(const abx_chunk_args* args, void* workspace, size_t workspace_bytes, abx_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* ABX_H_ */
