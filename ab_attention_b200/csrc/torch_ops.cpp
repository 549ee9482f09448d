// torch.ops.ab_attention: the PyTorch operator layer over the libabx C ABI.
//
// Replaces the reference's pybind module `ab_attention._C` (csrc/bindings.cpp:3-8,
// csrc/ops.h:5-8: `ibcs(q, k) -> scores`, `sip(scores, offsets, ids, logs)`) and
// the sparse prefill its FlashInfer adapter runs (ab_attention/flashinfer_backend.py:
// 164-242), as TORCH_LIBRARY operators callable from Python, C++ and TorchScript.
// Each operator checks its tensors (device, dtype, shape, contiguity) the way the
// reference's TORCH_CHECKs do, allocates outputs and workspaces with the caching
// allocator, and calls the extern "C" entry points of include/abx.h on the current
// CUDA stream; a nonzero status becomes a RuntimeError with libabx's message.
// Only CUDA kernels are registered: a CPU tensor finds no kernel and raises, so
// there is no silent fallback. Meta kernels give the output shapes to tracers.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <limits>
#include <optional>
#include <tuple>

#include "abx.h"

namespace {

constexpr int64_t kHeadDim = 128;
constexpr int64_t kQueryBlock = 128;

void check_status(int status, const char* what) {
    TORCH_CHECK(status == ABX_OK, what, " failed: ", abx_status_string(status), ": ", abx_last_error());
}

abx_stream_t stream_of(const at::Tensor& t) {
    return reinterpret_cast<abx_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void expect(const at::Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType dtype,
            const at::Tensor& like) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, " (got ", t.scalar_type(), ")");
    TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape, " (got ", t.sizes(), ")");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// [B, H, S, 128] or [BH, S, 128] -> (BH, S)
std::pair<int64_t, int64_t> heads_tokens(const at::Tensor& x, const char* name) {
    TORCH_CHECK(x.dim() == 3 || x.dim() == 4, name, " must be [B, H, S, 128] or [BH, S, 128]");
    TORCH_CHECK(x.size(-1) == kHeadDim, name, " must have head_dim 128");
    const int64_t bh = x.dim() == 4 ? x.size(0) * x.size(1) : x.size(0);
    return {bh, x.size(-2)};
}

int64_t rows_of(int64_t bh, int64_t seq) { return bh * ((seq + kQueryBlock - 1) / kQueryBlock); }

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
    // 256 bytes of slack: the caching allocator's blocks are 512-byte aligned, the
    // slack keeps a later alignment change from starving the layout
    return at::empty({bytes + 256}, like.options().dtype(at::kByte));
}

void* aligned256(const at::Tensor& ws) {
    const auto p = reinterpret_cast<uintptr_t>(ws.data_ptr());
    return reinterpret_cast<void*>((p + 255) & ~static_cast<uintptr_t>(255));
}

// `_C.ibcs(q, k) -> scores` (csrc/ibcs.cu:549-617): f32 [BH * ceil(S/128), S/4].
at::Tensor ibcs_cuda(const at::Tensor& q, const at::Tensor& k) {
    const auto [bh, seq] = heads_tokens(q, "q");
    expect(q, "q", q.sizes(), at::kBFloat16, q);
    expect(k, "k", q.sizes(), at::kBFloat16, q);
    c10::cuda::CUDAGuard guard(q.device());
    size_t bytes = 0;
    check_status(abx_ibcs_workspace_size(bh, seq, &bytes), "abx_ibcs_workspace_size");
    auto ws = workspace(static_cast<int64_t>(bytes), q);
    auto scores = at::empty({rows_of(bh, seq), seq / 4}, q.options().dtype(at::kFloat));
    check_status(abx_ibcs_scores(q.data_ptr(), k.data_ptr(), bh, seq, scores.data_ptr<float>(), aligned256(ws),
                                 bytes, stream_of(q)),
                 "abx_ibcs_scores");
    return scores;
}

// `_C.sip(scores, offsets, ids, logs)` (csrc/sip.cu:170-199): ids/logs written in place.
void sip_cuda(const at::Tensor& scores, const at::Tensor& offsets, at::Tensor ids, at::Tensor logs) {
    TORCH_CHECK(scores.dim() == 2 && ids.dim() == 2, "expected scores [rows, N] and ids/logs [rows, samples]");
    const int64_t rows = scores.size(0), population = scores.size(1), samples = ids.size(1);
    expect(scores, "scores", {rows, population}, at::kFloat, scores);
    expect(offsets, "offsets", {rows}, at::kFloat, scores);
    expect(ids, "ids", {rows, samples}, at::kInt, scores);
    expect(logs, "logs", {rows, samples}, at::kFloat, scores);
    c10::cuda::CUDAGuard guard(scores.device());
    check_status(abx_sip(scores.data_ptr<float>(), offsets.data_ptr<float>(), rows, population,
                         ids.data_ptr<int32_t>(), logs.data_ptr<float>(), samples, stream_of(scores)),
                 "abx_sip");
}

// build_plan's device work (ab_attention/attention.py:27-82) for given uniforms:
// (ids int32, log_weights f32) [rows, samples].
std::tuple<at::Tensor, at::Tensor> build_plan_cuda(const at::Tensor& q, const at::Tensor& k,
                                                   const at::Tensor& offsets, int64_t samples) {
    const auto [bh, seq] = heads_tokens(q, "q");
    const int64_t rows = rows_of(bh, seq);
    expect(q, "q", q.sizes(), at::kBFloat16, q);
    expect(k, "k", q.sizes(), at::kBFloat16, q);
    expect(offsets, "offsets", {rows}, at::kFloat, q);
    c10::cuda::CUDAGuard guard(q.device());
    size_t bytes = 0;
    check_status(abx_ibcs_workspace_size(bh, seq, &bytes), "abx_ibcs_workspace_size");
    auto ws = workspace(static_cast<int64_t>(bytes), q);
    auto ids = at::empty({rows, samples}, q.options().dtype(at::kInt));
    auto logw = at::empty({rows, samples}, q.options().dtype(at::kFloat));
    check_status(abx_build_plan(q.data_ptr(), k.data_ptr(), bh, seq, offsets.data_ptr<float>(), samples,
                                ids.data_ptr<int32_t>(), logw.data_ptr<float>(), aligned256(ws), bytes, stream_of(q)),
                 "abx_build_plan");
    return {ids, logw};
}

// The HT-weighted sparse prefill (flashinfer_backend.py:164-242 with the
// ABSipAttention shift, :30-58) over [BH, S, 128] q/k/v and a plan [rows,
// samples]: (o bf16 [BH, S, 128], base-2 lse f32 [BH, S]). Two adjacent query
// blocks per CTA when the shape pairs, one otherwise.
std::tuple<at::Tensor, at::Tensor> sparse_prefill_cuda(const at::Tensor& q, const at::Tensor& k,
                                                       const at::Tensor& v, const at::Tensor& ids,
                                                       const at::Tensor& log_weights) {
    TORCH_CHECK(q.dim() == 3, "q must be [batch*heads, tokens, 128]");
    const int64_t bh = q.size(0), seq = q.size(1);
    TORCH_CHECK(ids.dim() == 2, "ids must be [rows, samples]");
    const int64_t samples = ids.size(1), rows = rows_of(bh, seq);
    expect(q, "q", {bh, seq, kHeadDim}, at::kBFloat16, q);
    expect(k, "k", {bh, seq, kHeadDim}, at::kBFloat16, q);
    expect(v, "v", {bh, seq, kHeadDim}, at::kBFloat16, q);
    expect(ids, "ids", {rows, samples}, at::kInt, q);
    expect(log_weights, "log_weights", {rows, samples}, at::kFloat, q);
    c10::cuda::CUDAGuard guard(q.device());
    auto o = at::empty_like(q);
    auto lse = at::empty({bh, seq}, q.options().dtype(at::kFloat));
    size_t bytes = 0;
    check_status(abx_prefill_workspace_size(bh, seq, samples, 0, &bytes), "abx_prefill_workspace_size");
    if (bytes > 0) {
        auto ws = workspace(static_cast<int64_t>(bytes), q);
        check_status(abx_sparse_prefill_paired(q.data_ptr(), k.data_ptr(), v.data_ptr(), bh, seq,
                                               ids.data_ptr<int32_t>(), log_weights.data_ptr<float>(), samples,
                                               nullptr, nullptr, 0, o.data_ptr(), lse.data_ptr<float>(),
                                               aligned256(ws), bytes, stream_of(q)),
                     "abx_sparse_prefill_paired");
    } else {
        check_status(abx_sparse_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), bh, seq, ids.data_ptr<int32_t>(),
                                        log_weights.data_ptr<float>(), samples, nullptr, nullptr, 0, o.data_ptr(),
                                        lse.data_ptr<float>(), stream_of(q)),
                     "abx_sparse_prefill");
    }
    return {o, lse};
}

// ---- streaming operators: rotary positions, cache append, chunk and window attention -------
// Argument errors raise ValueError. The checks are shared with the Meta kernels.

// A new CUDA tensor on `like`'s device, without another trip through the dispatcher (half a microsecond a tensor).
at::Tensor fresh(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(size, dtype, like.device(), std::nullopt));
}

int dtype_code(const at::Tensor& t, const char* name, bool f32 = false) {
    if (t.scalar_type() == at::kBFloat16) return ABX_BF16;
    if (t.scalar_type() == at::kHalf) return ABX_FP16;
    TORCH_CHECK_VALUE(f32 && t.scalar_type() == at::kFloat, name, " must be bfloat16", f32 ? ", float16 or float32" : " or float16",
                      " (got ", t.scalar_type(), ")");
    return ABX_F32;
}

void like(const at::Tensor& t, const char* name, const at::Tensor& other, at::ScalarType dtype) {
    TORCH_CHECK_VALUE(t.device() == other.device(), name, " must be on ", other.device(), " (got ", t.device(), ")");
    TORCH_CHECK_VALUE(t.scalar_type() == dtype, name, " must be ", dtype, " (got ", t.scalar_type(), ")");
}

void index_vector(const at::Tensor& t, const char* name, const at::Tensor& other, int64_t size) {
    like(t, name, other, at::kInt);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == size, name, " must be int32 [", size, "] (got ", t.sizes(), ")");
    TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}

// Rows of 128 contiguous elements that each start on a 16-byte boundary. `packed`
// also wants distinct rows (tensor maps and outputs cannot repeat one by a zero stride).
bool rows_fit(const at::Tensor& t, bool packed) {
    const int64_t e = t.element_size();
    if (t.stride(-1) != 1 || (!t.is_meta() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0)) return false;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) {
        if (t.size(d) <= 1) continue;
        const int64_t s = t.stride(d);
        if (s < 0 || s * e % 16 != 0 || (packed && s == 0) || s * e >= (int64_t(1) << 40)) return false;
    }
    return true;
}

void expect_rows(const at::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(rows_fit(t, true), name, " must have contiguous 16-byte aligned rows of 128 elements");
}

at::Tensor as_rows(const at::Tensor& t, bool packed) { return rows_fit(t, packed) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Strides (outer, head, token) of the dims given; a dim of one element counts 0.
void strides_of(const at::Tensor& t, int64_t (&out)[3], int outer, int head, int token) {
    const int dims[3] = {outer, head, token};
    for (int i = 0; i < 3; ++i) out[i] = dims[i] < 0 || t.size(dims[i]) <= 1 ? 0 : t.stride(dims[i]);
}

void check_axes(at::IntArrayRef sections, double theta) {
    int64_t dims = 0;
    TORCH_CHECK_VALUE(sections.size() >= 1 && sections.size() <= 4, "sections must name 1 to 4 axes (got ", sections.size(), ")");
    for (int64_t s : sections) {
        TORCH_CHECK_VALUE(s >= 0 && s % 2 == 0, "sections must be even and not negative (got ", sections, ")");
        dims += s;
    }
    TORCH_CHECK_VALUE(dims == kHeadDim, "sections must sum to 128 (got ", sections, ")");
    TORCH_CHECK_VALUE(theta > 0 && theta < 1e300, "theta must be positive and finite");
}

void set_axes(abx_rotary_args& r, at::IntArrayRef sections, double theta, bool shared, bool halves, bool inverse) {
    r.axes = static_cast<int32_t>(sections.size());
    for (size_t i = 0; i < sections.size(); ++i) r.sections[i] = static_cast<int32_t>(sections[i]);
    r.theta = theta;
    r.shared = shared;
    r.halves = halves;
    r.inverse = inverse;
}

void check_rotary(const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions,
                  at::IntArrayRef sections, double theta) {
    TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == kHeadDim, "q must be [B,H,N,128] (got ", q.sizes(), ")");
    dtype_code(q, "q", true);
    if (k) {
        like(*k, "k", q, q.scalar_type());
        TORCH_CHECK_VALUE(k->dim() == 4 && k->size(0) == q.size(0) && k->size(2) == q.size(2) && k->size(3) == kHeadDim,
                          "k must be [B,Hk,N,128] with q's batch and tokens (got ", k->sizes(), ")");
    }
    check_axes(sections, theta);
    like(positions, "positions", q, at::kInt);
    const int64_t axes = static_cast<int64_t>(sections.size());
    TORCH_CHECK_VALUE((positions.dim() == 2 && positions.size(0) == q.size(2) && positions.size(1) == axes) ||
                          (positions.dim() == 3 && positions.size(0) == q.size(0) && positions.size(1) == q.size(2) &&
                           positions.size(2) == axes),
                      "positions must be int32 [N,", axes, "] or [B,N,", axes, "] (got ", positions.sizes(), ")");
}

std::tuple<at::Tensor, at::Tensor> rotary_cuda(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                               const at::Tensor& positions, at::IntArrayRef sections, double theta,
                                               bool shared, bool halves, bool inverse) {
    check_rotary(q, k, positions, sections, theta);
    c10::cuda::CUDAGuard guard(q.device());
    auto q_out = fresh(q.sizes(), q.scalar_type(), q);
    auto k_out = fresh(k ? k->sizes() : at::IntArrayRef({0}), q.scalar_type(), q);
    abx_rotary_args r{};
    r.dtype = dtype_code(q, "q", true);
    set_axes(r, sections, theta, shared, halves, inverse);
    const auto where = positions.contiguous();
    r.positions = where.data_ptr<int32_t>();
    r.positions_batch = where.dim() == 3 ? where.size(1) * where.size(2) : 0;
    r.batch = q.size(0);
    r.tokens = q.size(2);
    at::Tensor qr, kr;
    if (q.numel() > 0) {
        qr = as_rows(q, false);
        r.q = qr.data_ptr();
        r.q_out = q_out.data_ptr();
        r.heads = q.size(1);
        strides_of(qr, r.q_stride, 0, 1, 2);
        strides_of(q_out, r.q_out_stride, 0, 1, 2);
    }
    if (k && k->numel() > 0) {
        kr = as_rows(*k, false);
        r.k = kr.data_ptr();
        r.k_out = k_out.data_ptr();
        r.kv_heads = k->size(1);
        strides_of(kr, r.k_stride, 0, 1, 2);
        strides_of(k_out, r.k_out_stride, 0, 1, 2);
    }
    if (r.q || r.k) check_status(abx_rotary(&r, stream_of(q)), "abx_rotary");
    return {q_out, k_out};
}

void check_cache(const at::Tensor& keys, const at::Tensor& values) {
    TORCH_CHECK_VALUE(keys.dim() == 4 && keys.size(3) == kHeadDim,
                      "cache keys must be [pages, kv_heads, page_size, 128] (got ", keys.sizes(), ")");
    dtype_code(keys, "cache keys");
    like(values, "cache values", keys, keys.scalar_type());
    TORCH_CHECK_VALUE(values.sizes() == keys.sizes(), "cache values must have the keys' shape (got ", values.sizes(), ")");
    TORCH_CHECK_VALUE(keys.numel() > 0, "the cache must have pages");
    const int64_t page = keys.size(2);
    TORCH_CHECK_VALUE(page == 16 || page == 32 || page == 64 || (page > 0 && page % 128 == 0),
                      "page size must be 16, 32, 64 or a multiple of 128 (got ", page, ")");
    expect_rows(keys, "cache keys");
    expect_rows(values, "cache values");
}

void check_batch(const at::Tensor& keys, const at::Tensor& page_table, const at::Tensor& starts, const at::Tensor& lengths) {
    like(page_table, "page_table", keys, at::kInt);
    TORCH_CHECK_VALUE(page_table.dim() == 2 && page_table.size(1) > 0 && page_table.is_contiguous(),
                      "page_table must be contiguous int32 [sequences, pages] (got ", page_table.sizes(), ")");
    index_vector(starts, "starts", keys, page_table.size(0) + 1);
    index_vector(lengths, "lengths", keys, page_table.size(0));
}

void check_append(const at::Tensor& keys, const at::Tensor& values, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& page_table, const at::Tensor& starts, const at::Tensor& lengths,
                  const std::optional<at::Tensor>& q, const std::optional<at::Tensor>& positions,
                  at::IntArrayRef sections, double theta) {
    check_cache(keys, values);
    check_batch(keys, page_table, starts, lengths);
    for (const auto* t : {&k, &v}) {
        const char* name = t == &k ? "k" : "v";
        like(*t, name, keys, keys.scalar_type());
        TORCH_CHECK_VALUE(t->dim() == 3 && t->size(0) == k.size(0) && t->size(1) == keys.size(1) && t->size(2) == kHeadDim,
                          name, " must be [tokens, ", keys.size(1), ", 128] (got ", t->sizes(), ")");
    }
    TORCH_CHECK_VALUE(!q || positions, "q is turned with positions: give both");
    if (q) {
        like(*q, "q", keys, keys.scalar_type());
        TORCH_CHECK_VALUE(q->dim() == 3 && q->size(0) == k.size(0) && q->size(2) == kHeadDim,
                          "q must be [tokens, heads, 128] (got ", q->sizes(), ")");
    }
    if (positions) {
        check_axes(sections, theta);
        like(*positions, "positions", keys, at::kInt);
        TORCH_CHECK_VALUE(positions->dim() == 2 && positions->size(0) == k.size(0) &&
                              positions->size(1) == static_cast<int64_t>(sections.size()),
                          "positions must be int32 [tokens, ", sections.size(), "] (got ", positions->sizes(), ")");
    }
}

at::Tensor append_cuda(at::Tensor keys, at::Tensor values, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& page_table, const at::Tensor& starts, const at::Tensor& lengths,
                       const std::optional<at::Tensor>& q, const std::optional<at::Tensor>& positions,
                       at::IntArrayRef sections, double theta, bool shared, bool halves) {
    check_append(keys, values, k, v, page_table, starts, lengths, q, positions, sections, theta);
    c10::cuda::CUDAGuard guard(keys.device());
    auto q_out = fresh(q ? q->sizes() : at::IntArrayRef({0}), keys.scalar_type(), keys);
    if (k.size(0) == 0 || page_table.size(0) == 0) {
        TORCH_CHECK_VALUE(k.size(0) == 0, "tokens without a sequence");
        return q_out;
    }
    abx_rotary_args r{};
    r.dtype = dtype_code(keys, "cache keys");
    at::Tensor where, qr;
    if (positions) {
        set_axes(r, sections, theta, shared, halves, false);
        where = positions->contiguous();
        r.positions = where.data_ptr<int32_t>();
    }
    r.batch = 1;
    r.tokens = k.size(0);
    if (q && q->numel() > 0) {
        qr = as_rows(*q, false);
        r.q = qr.data_ptr();
        r.q_out = q_out.data_ptr();
        r.heads = q->size(1);
        strides_of(qr, r.q_stride, -1, 1, 0);
        strides_of(q_out, r.q_out_stride, -1, 1, 0);
    }
    const auto kr = as_rows(k, false), vr = as_rows(v, false);
    r.k = kr.data_ptr();
    r.v = vr.data_ptr();
    r.k_out = keys.data_ptr();
    r.v_out = values.data_ptr();
    r.kv_heads = keys.size(1);
    strides_of(kr, r.k_stride, -1, 1, 0);
    strides_of(vr, r.v_stride, -1, 1, 0);
    strides_of(keys, r.k_out_stride, 0, 1, 2);
    strides_of(values, r.v_out_stride, 0, 1, 2);
    r.starts = starts.data_ptr<int32_t>();
    r.lengths = lengths.data_ptr<int32_t>();
    r.page_table = page_table.data_ptr<int32_t>();
    r.sequences = page_table.size(0);
    r.table_width = page_table.size(1);
    r.page_size = keys.size(2);
    r.pages = keys.size(0);
    check_status(abx_rotary(&r, stream_of(keys)), "abx_rotary");
    return q_out;
}

void check_rule(int64_t window, int64_t sinks, int64_t block) {
    TORCH_CHECK_VALUE(window >= 0, "window must be positive, or None");
    TORCH_CHECK_VALUE(sinks >= 0, "sinks must not be negative");
    TORCH_CHECK_VALUE(block >= 1, "block must be positive");
}

void attend(abx_chunk_args& c, const at::Tensor& q) {
    size_t bytes = 0;
    check_status(abx_chunk_workspace_size(&c, &bytes), "abx_chunk_workspace_size");
    at::Tensor ws;
    if (bytes > 0) ws = fresh({static_cast<int64_t>(bytes) + 256}, at::kByte, q);
    check_status(abx_chunk_attention(&c, bytes > 0 ? aligned256(ws) : nullptr, bytes, stream_of(q)), "abx_chunk_attention");
}

void check_chunk(const at::Tensor& q, const at::Tensor& keys, const at::Tensor& values, const at::Tensor& page_table,
                 const at::Tensor& starts, const at::Tensor& lengths, int64_t longest, int64_t window, int64_t sinks,
                 int64_t block, const at::Tensor& out, const std::optional<at::Tensor>& lse) {
    check_cache(keys, values);
    check_batch(keys, page_table, starts, lengths);
    like(q, "q", keys, keys.scalar_type());
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == kHeadDim && q.size(1) > 0 && q.size(1) % keys.size(1) == 0,
                      "q must be [tokens, heads, 128] with heads a multiple of ", keys.size(1), " (got ", q.sizes(), ")");
    check_rule(window, sinks, block);
    TORCH_CHECK_VALUE(longest >= 1 || q.size(0) == 0, "longest must be positive (got ", longest, ")");
    like(out, "out", q, q.scalar_type());
    TORCH_CHECK_VALUE(out.sizes() == q.sizes(), "out must have q's shape (got ", out.sizes(), ")");
    expect_rows(out, "out");
    if (lse) {
        like(*lse, "lse", q, at::kFloat);
        TORCH_CHECK_VALUE(lse->dim() == 2 && lse->size(0) == q.size(0) && lse->size(1) == q.size(1),
                          "lse must be float32 [tokens, heads] (got ", lse->sizes(), ")");
    }
}

void chunk_attention_out_cuda(const at::Tensor& q, const at::Tensor& keys, const at::Tensor& values,
                          const at::Tensor& page_table, const at::Tensor& starts, const at::Tensor& lengths,
                          int64_t longest, int64_t window, int64_t sinks, int64_t block, at::Tensor out,
                          std::optional<at::Tensor> lse) {
    check_chunk(q, keys, values, page_table, starts, lengths, longest, window, sinks, block, out, lse);
    if (q.numel() == 0 || page_table.size(0) == 0) return;
    c10::cuda::CUDAGuard guard(q.device());
    const auto qr = as_rows(q, false);
    abx_chunk_args c{};
    c.dtype = dtype_code(q, "q");
    c.q = qr.data_ptr();
    c.k = keys.data_ptr();
    c.v = values.data_ptr();
    c.o = out.data_ptr();
    strides_of(qr, c.q_stride, -1, 1, 0);
    strides_of(keys, c.k_stride, 0, 1, 2);
    strides_of(values, c.v_stride, 0, 1, 2);
    strides_of(out, c.o_stride, -1, 1, 0);
    if (lse) {
        c.lse = lse->data_ptr<float>();
        strides_of(*lse, c.lse_stride, -1, 1, 0);
    }
    c.sequences = page_table.size(0);
    c.tokens = q.size(0);
    c.longest = std::min(longest, q.size(0));
    c.heads = q.size(1);
    c.kv_heads = keys.size(1);
    c.starts = starts.data_ptr<int32_t>();
    c.lengths = lengths.data_ptr<int32_t>();
    c.page_table = page_table.data_ptr<int32_t>();
    c.table_width = page_table.size(1);
    c.page_size = keys.size(2);
    c.pages = keys.size(0);
    c.window = window;
    c.sinks = sinks;
    c.block = block;
    attend(c, q);
}

std::tuple<at::Tensor, at::Tensor> chunk_results(const at::Tensor& q, bool lse) {
    TORCH_CHECK_VALUE(q.dim() == 3, "q must be [tokens, heads, 128] (got ", q.sizes(), ")");
    if (q.is_meta())
        return {at::empty(q.sizes(), q.options()), at::empty({lse ? q.size(0) : 0, q.size(1)}, q.options().dtype(at::kFloat))};
    return {fresh(q.sizes(), q.scalar_type(), q), fresh({lse ? q.size(0) : 0, q.size(1)}, at::kFloat, q)};
}

std::tuple<at::Tensor, at::Tensor> chunk_attention_cuda(const at::Tensor& q, const at::Tensor& keys, const at::Tensor& values,
                                                        const at::Tensor& page_table, const at::Tensor& starts,
                                                        const at::Tensor& lengths, int64_t longest, int64_t window,
                                                        int64_t sinks, int64_t block, bool want_lse) {
    auto [out, lse] = chunk_results(q, want_lse);
    chunk_attention_out_cuda(q, keys, values, page_table, starts, lengths, longest, window, sinks, block, out,
                             want_lse ? std::optional<at::Tensor>(lse) : std::nullopt);
    return {out, lse};
}

void check_window(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window, int64_t sinks, int64_t block) {
    TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == kHeadDim, "q must be [B,H,N,128] (got ", q.sizes(), ")");
    dtype_code(q, "q");
    like(k, "k", q, q.scalar_type());
    like(v, "v", q, q.scalar_type());
    TORCH_CHECK_VALUE(k.dim() == 4 && k.size(0) == q.size(0) && k.size(3) == kHeadDim && k.size(1) > 0 &&
                          q.size(1) % k.size(1) == 0,
                      "k must be [B,Hk,Nk,128] with Hk dividing q's heads (got ", k.sizes(), ")");
    TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "v must have k's shape (got ", v.sizes(), ")");
    check_rule(window, sinks, block);
}

std::tuple<at::Tensor, at::Tensor> window_attention_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                         int64_t window, int64_t sinks, int64_t block) {
    check_window(q, k, v, window, sinks, block);
    c10::cuda::CUDAGuard guard(q.device());
    auto out = fresh(q.sizes(), q.scalar_type(), q);
    auto lse = fresh({q.size(0), q.size(1), q.size(2)}, at::kFloat, q);
    if (q.numel() == 0) return {out, lse};
    if (k.numel() == 0) return {out.zero_(), lse.fill_(-std::numeric_limits<float>::infinity())};
    const auto qr = as_rows(q, false), kr = as_rows(k, true), vr = as_rows(v, true);
    abx_chunk_args c{};
    c.dtype = dtype_code(q, "q");
    c.q = qr.data_ptr();
    c.k = kr.data_ptr();
    c.v = vr.data_ptr();
    c.o = out.data_ptr();
    c.lse = lse.data_ptr<float>();
    strides_of(qr, c.q_stride, 0, 1, 2);
    strides_of(kr, c.k_stride, 0, 1, 2);
    strides_of(vr, c.v_stride, 0, 1, 2);
    strides_of(out, c.o_stride, 0, 1, 2);
    strides_of(lse, c.lse_stride, 0, 1, 2);
    c.sequences = q.size(0);
    c.tokens = c.longest = q.size(2);
    c.keys = k.size(2);
    c.heads = q.size(1);
    c.kv_heads = k.size(1);
    c.window = window;
    c.sinks = sinks;
    c.block = block;
    attend(c, q);
    return {out, lse};
}

// ---- shapes for tracers (no data, no kernels) ----------------------------------------

std::tuple<at::Tensor, at::Tensor> rotary_meta(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                               const at::Tensor& positions, at::IntArrayRef sections, double theta, bool,
                                               bool, bool) {
    check_rotary(q, k, positions, sections, theta);
    return {at::empty(q.sizes(), q.options()), k ? at::empty(k->sizes(), k->options()) : at::empty({0}, q.options())};
}

at::Tensor append_meta(at::Tensor keys, at::Tensor values, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& page_table, const at::Tensor& starts, const at::Tensor& lengths,
                       const std::optional<at::Tensor>& q, const std::optional<at::Tensor>& positions,
                       at::IntArrayRef sections, double theta, bool, bool) {
    check_append(keys, values, k, v, page_table, starts, lengths, q, positions, sections, theta);
    return q ? at::empty(q->sizes(), q->options()) : at::empty({0}, keys.options());
}

void chunk_attention_out_meta(const at::Tensor& q, const at::Tensor& keys, const at::Tensor& values,
                          const at::Tensor& page_table, const at::Tensor& starts, const at::Tensor& lengths,
                          int64_t longest, int64_t window, int64_t sinks, int64_t block, at::Tensor out,
                          std::optional<at::Tensor> lse) {
    check_chunk(q, keys, values, page_table, starts, lengths, longest, window, sinks, block, out, lse);
}

std::tuple<at::Tensor, at::Tensor> chunk_attention_meta(const at::Tensor& q, const at::Tensor& keys, const at::Tensor& values,
                                                        const at::Tensor& page_table, const at::Tensor& starts,
                                                        const at::Tensor& lengths, int64_t longest, int64_t window,
                                                        int64_t sinks, int64_t block, bool want_lse) {
    auto [out, lse] = chunk_results(q, want_lse);
    check_chunk(q, keys, values, page_table, starts, lengths, longest, window, sinks, block, out,
                want_lse ? std::optional<at::Tensor>(lse) : std::nullopt);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> window_attention_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                         int64_t window, int64_t sinks, int64_t block) {
    check_window(q, k, v, window, sinks, block);
    return {at::empty(q.sizes(), q.options()), at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

at::Tensor ibcs_meta(const at::Tensor& q, const at::Tensor& k) {
    const auto [bh, seq] = heads_tokens(q, "q");
    return at::empty({rows_of(bh, seq), seq / 4}, q.options().dtype(at::kFloat));
}

void sip_meta(const at::Tensor&, const at::Tensor&, at::Tensor, at::Tensor) {}

std::tuple<at::Tensor, at::Tensor> build_plan_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                   int64_t samples) {
    const auto [bh, seq] = heads_tokens(q, "q");
    const int64_t rows = rows_of(bh, seq);
    return {at::empty({rows, samples}, q.options().dtype(at::kInt)),
            at::empty({rows, samples}, q.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor> sparse_prefill_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                       const at::Tensor&, const at::Tensor&) {
    return {at::empty_like(q), at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}

}  // namespace

TORCH_LIBRARY(ab_attention, m) {
    m.def("ibcs(Tensor q, Tensor k) -> Tensor");
    m.def("sip(Tensor scores, Tensor offsets, Tensor(a!) ids, Tensor(b!) logs) -> ()");
    m.def("build_plan(Tensor q, Tensor k, Tensor offsets, int samples) -> (Tensor, Tensor)");
    m.def("sparse_prefill(Tensor q, Tensor k, Tensor v, Tensor ids, Tensor log_weights) -> (Tensor, Tensor)");
    m.def("rotary(Tensor q, Tensor? k, Tensor positions, int[] sections, float theta, bool shared, bool halves, "
          "bool inverse) -> (Tensor, Tensor)");
    m.def("append(Tensor(a!) keys, Tensor(b!) values, Tensor k, Tensor v, Tensor page_table, Tensor starts, "
          "Tensor lengths, Tensor? q, Tensor? positions, int[] sections, float theta, bool shared, bool halves) -> Tensor");
    m.def("chunk_attention(Tensor q, Tensor keys, Tensor values, Tensor page_table, Tensor starts, Tensor lengths, "
          "int longest, int window, int sinks, int block, bool lse) -> (Tensor, Tensor)");
    m.def("chunk_attention_out(Tensor q, Tensor keys, Tensor values, Tensor page_table, Tensor starts, Tensor lengths, "
          "int longest, int window, int sinks, int block, Tensor(a!) out, Tensor(b!)? lse) -> ()");
    m.def("window_attention(Tensor q, Tensor k, Tensor v, int window, int sinks, int block) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(ab_attention, CUDA, m) {
    m.impl("ibcs", &ibcs_cuda);
    m.impl("sip", &sip_cuda);
    m.impl("build_plan", &build_plan_cuda);
    m.impl("sparse_prefill", &sparse_prefill_cuda);
    m.impl("rotary", &rotary_cuda);
    m.impl("append", &append_cuda);
    m.impl("chunk_attention", &chunk_attention_cuda);
    m.impl("chunk_attention_out", &chunk_attention_out_cuda);
    m.impl("window_attention", &window_attention_cuda);
}

TORCH_LIBRARY_IMPL(ab_attention, Meta, m) {
    m.impl("ibcs", &ibcs_meta);
    m.impl("sip", &sip_meta);
    m.impl("build_plan", &build_plan_meta);
    m.impl("sparse_prefill", &sparse_prefill_meta);
    m.impl("rotary", &rotary_meta);
    m.impl("append", &append_meta);
    m.impl("chunk_attention", &chunk_attention_meta);
    m.impl("chunk_attention_out", &chunk_attention_out_meta);
    m.impl("window_attention", &window_attention_meta);
}

// No gradients, as everywhere in the package: the streaming operators pass the autograd keys by, which
// also spares their callers a no_grad block.
TORCH_LIBRARY_IMPL(ab_attention, Autograd, m) {
    for (const char* name : {"rotary", "append", "chunk_attention", "chunk_attention_out", "window_attention"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}
