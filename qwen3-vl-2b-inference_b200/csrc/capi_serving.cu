// C ABI of the operators that serve drafted and multimodal tokens over the
// paged cache: argument checks, then one launcher each (serving.cuh).
#include <cstring>
#include "serving.cuh"

namespace {
bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool al4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
// Bytes of a float type this file's operators take; 0 for any other.
size_t float_bytes(int dtype) {
    switch (dtype) {
    case QVL_DTYPE_FP32: return 4;
    case QVL_DTYPE_FP16:
    case QVL_DTYPE_BF16: return 2;
    default: return 0;
    }
}
// Rows of `width` elements `stride` elements apart, read in 16-byte pieces.
bool rows_ok(const void *p, size_t stride, size_t width, size_t bytes) {
    return p && al16(p) && stride >= width && stride <= (size_t)INT32_MAX && stride * bytes % 16 == 0;
}
bool dims_ok(const qvl_attn_dims *d) {
    return d && d->num_heads > 0 && d->num_kv_heads > 0 && d->num_heads % d->num_kv_heads == 0 && d->page_size >= 16 &&
           d->page_size % 16 == 0 && d->max_pages_per_seq > 0;
}
}  // namespace

extern "C" {

int qvl_plan_pages(const int32_t *old_lengths, const int32_t *new_lengths, size_t n_seqs, int32_t *page_table,
                   int page_size, int max_pages_per_seq, int32_t *free_pages, const int32_t *free_count,
                   size_t capacity, int32_t *free_count_out, int32_t *missing, int32_t *starts, int32_t *seq_ids,
                   int32_t *positions, int32_t *slots, size_t max_tokens, void *stream) {
    if (!old_lengths || !new_lengths || !page_table || !free_pages || !free_count || !free_count_out || !missing ||
        !starts || (max_tokens && (!seq_ids || !positions || !slots)))
        return QVL_ERR_INVALID;
    if (n_seqs == 0 || page_size <= 0 || max_pages_per_seq <= 0 || free_count == free_count_out) return QVL_ERR_INVALID;
    // (the kernel's stretches of tokens end up to 4704 * 32 past the last one)
    if (capacity > (size_t)INT32_MAX || max_tokens > (size_t)INT32_MAX - (1u << 18)) return QVL_ERR_INVALID;
    const void *p[] = {old_lengths, new_lengths, page_table, free_pages, free_count, free_count_out,
                       missing,     starts,      seq_ids,    positions,  slots};
    for (const void *x : p)
        if (!al4(x)) return QVL_ERR_INVALID;
    if (n_seqs > (size_t)qvl::kPlanMaxSeqs) return QVL_ERR_UNSUPPORTED;
    const qvl::PlanArgs a{old_lengths, new_lengths,    (int)n_seqs, page_table, page_size, max_pages_per_seq,
                          free_pages,  free_count,     (int)capacity, free_count_out, missing, starts,
                          seq_ids,     positions,      slots,       (int)max_tokens};
    QVL_CUDA_TRY(qvl::launch_plan_pages(a, (cudaStream_t)stream));
    return QVL_OK;
}

int qvl_qknorm_mrope_kv_append(const void *q, const void *k, const void *v, int dtype, size_t q_stride, size_t k_stride,
                               size_t v_stride, void *q_out, void *k_pages, void *v_pages, int kv_dtype,
                               size_t num_pages, const int32_t *slots, const int32_t *positions, size_t pos_stride,
                               int n_axes, const int32_t *axes, size_t n_tokens, const float *rope_cos,
                               const float *rope_sin, const void *q_norm_w, const float *q_norm_s,
                               const void *k_norm_w, const float *k_norm_s, int norm_dtype, size_t norm_group,
                               float eps, const qvl_attn_dims *dims, void *stream) {
    if (!dims_ok(dims) || dims->head_dim <= 0 || dims->max_pos <= 0) return QVL_ERR_INVALID;
    const size_t b = float_bytes(dtype);
    const int D = dims->head_dim;
    if (!b || (kv_dtype != QVL_DTYPE_FP16 && kv_dtype != QVL_DTYPE_BF16) || (D != 64 && D != 128 && D != 256))
        return QVL_ERR_UNSUPPORTED;
    if (n_tokens == 0) return QVL_OK;
    if (!q_out || !k_pages || !v_pages || !slots || !positions || !axes || !rope_cos || !rope_sin)
        return QVL_ERR_INVALID;
    if (n_axes < 1 || n_axes > 8 || n_tokens > (1u << 26) || pos_stride < n_tokens || !(eps >= 0.0f) || num_pages == 0 ||
        num_pages > (size_t)INT32_MAX / dims->page_size)
        return QVL_ERR_INVALID;
    const size_t NH = dims->num_heads, NKV = dims->num_kv_heads;
    if (!rows_ok(q, q_stride, NH * D, b) || !rows_ok(k, k_stride, NKV * D, b) || !rows_ok(v, v_stride, NKV * D, b) ||
        !al16(q_out) || !al16(k_pages) || !al16(v_pages) || !al4(slots) || !al4(positions) || !al4(axes) ||
        !al4(rope_cos) || !al4(rope_sin))
        return QVL_ERR_INVALID;
    if (!q_norm_w != !k_norm_w) return QVL_ERR_INVALID;
    if (q_norm_w) {
        if (norm_dtype == QVL_DTYPE_INT8) {
            if (!q_norm_s || !k_norm_s || norm_group == 0 || D % norm_group) return QVL_ERR_INVALID;
        } else if (!float_bytes(norm_dtype)) {
            return QVL_ERR_UNSUPPORTED;
        }
        const uintptr_t m = norm_dtype == QVL_DTYPE_INT8 ? 0 : float_bytes(norm_dtype) - 1;
        if (((uintptr_t)q_norm_w | (uintptr_t)k_norm_w) & m) return QVL_ERR_INVALID;
        if (!al4(q_norm_s) || !al4(k_norm_s)) return QVL_ERR_INVALID;
    }
    qvl::MropeArgs a{};
    a.q = q; a.k = k; a.v = v;
    a.q_stride = (long)q_stride; a.k_stride = (long)k_stride; a.v_stride = (long)v_stride;
    a.q_out = q_out; a.k_pages = k_pages; a.v_pages = v_pages;
    a.slots = slots; a.positions = positions; a.axes = axes; a.pos_stride = (long)pos_stride;
    a.cos_t = rope_cos; a.sin_t = rope_sin;
    a.qn = {q_norm_w, q_norm_s, (int)norm_group};
    a.kn = {k_norm_w, k_norm_s, (int)norm_group};
    a.eps = eps;
    a.T = (int)n_tokens; a.NH = (int)NH; a.NKV = (int)NKV; a.D = D; a.P = dims->page_size;
    a.max_pos = dims->max_pos; a.n_axes = n_axes;
    a.num_slots = (long)num_pages * dims->page_size;
    a.dtype = dtype; a.kv_dtype = kv_dtype; a.w_dtype = norm_dtype;
    QVL_CUDA_TRY(qvl::launch_mrope_append(a, (cudaStream_t)stream));
    return QVL_OK;
}

size_t qvl_tree_attention_workspace_bytes(size_t n_seqs, size_t n_rows, int max_ctx, int max_nodes,
                                          const qvl_attn_dims *dims) {
    if (!dims_ok(dims) || n_seqs == 0 || n_seqs > 65535 || n_rows > (1u << 26) || max_ctx <= 0 || max_nodes <= 0 ||
        max_nodes > qvl::kTreeMaxNodes || (dims->head_dim != 64 && dims->head_dim != 128))
        return 0;
    return qvl::tree_workspace_bytes(dims->head_dim);
}

int qvl_tree_attention(const void *q, int dtype, size_t q_stride, const void *k_pages, const void *v_pages,
                       int kv_dtype, size_t num_pages, const int32_t *page_table, const int32_t *ctx_lens,
                       const int32_t *starts, const int32_t *parents, size_t n_seqs, size_t n_rows, int max_ctx,
                       int max_nodes, float scale, void *out, const qvl_attn_dims *dims, void *workspace,
                       size_t workspace_bytes, void *stream) {
    if (!dims_ok(dims) || dims->head_dim <= 0) return QVL_ERR_INVALID;
    const size_t b = float_bytes(dtype);
    const int D = dims->head_dim;
    // the matrix products take query and cache in one 16-bit type; fp32
    // queries over an fp16 cache go as a sum of two fp16 values
    const bool types = (kv_dtype == QVL_DTYPE_FP16 && (dtype == QVL_DTYPE_FP16 || dtype == QVL_DTYPE_FP32)) ||
                       (kv_dtype == QVL_DTYPE_BF16 && dtype == QVL_DTYPE_BF16);
    if (!types || (D != 64 && D != 128) || max_nodes > qvl::kTreeMaxNodes) return QVL_ERR_UNSUPPORTED;
    // the heads of a key head are more than 128: more than a tile of rows
    if (dims->num_heads / dims->num_kv_heads > 128) return QVL_ERR_UNSUPPORTED;
    if (n_rows == 0) return QVL_OK;
    if (!k_pages || !v_pages || !page_table || !ctx_lens || !starts || !parents || !out) return QVL_ERR_INVALID;
    const size_t NH = dims->num_heads;
    if (n_seqs == 0 || n_seqs > 65535 || n_rows > (1u << 26) || max_ctx <= 0 || max_nodes <= 0 || num_pages == 0 ||
        num_pages > (size_t)INT32_MAX || !(scale == scale))
        return QVL_ERR_INVALID;
    // TMA coordinates of the cache's rows are 32-bit
    if (num_pages * (size_t)dims->num_kv_heads > (size_t)INT32_MAX / dims->page_size) return QVL_ERR_UNSUPPORTED;
    if (dims->num_kv_heads > 65535) return QVL_ERR_UNSUPPORTED;
    if (!rows_ok(q, q_stride, NH * D, b)) return QVL_ERR_INVALID;
    if (!al16(k_pages) || !al16(v_pages) || !al16(out) || !al4(page_table) || !al4(ctx_lens) || !al4(starts) ||
        !al4(parents))
        return QVL_ERR_INVALID;
    if (!workspace || workspace_bytes < qvl::tree_workspace_bytes(D) || ((uintptr_t)workspace & 255))
        return QVL_ERR_WORKSPACE;
    qvl::TreeArgs a{};
    a.q = q; a.q_stride = (long)q_stride; a.k_pages = k_pages; a.v_pages = v_pages; a.num_pages = (long)num_pages;
    a.table = page_table; a.ctx_lens = ctx_lens; a.starts = starts; a.parents = parents;
    a.S = (int)n_seqs; a.T = (int)n_rows; a.max_ctx = max_ctx; a.max_nodes = max_nodes; a.scale = scale; a.out = out;
    a.NH = dims->num_heads; a.NKV = dims->num_kv_heads; a.D = D; a.P = dims->page_size;
    a.maxp = dims->max_pages_per_seq; a.dtype = dtype; a.kv_dtype = kv_dtype; a.workspace = workspace;
    QVL_CUDA_TRY(qvl::launch_tree_attention(a, (cudaStream_t)stream));
    return QVL_OK;
}

int qvl_token_logprobs(const void *logits, int dtype, size_t stride, const int32_t *tokens, size_t n_rows, size_t vocab,
                       int top_k, float *logprobs, float *entropy, int32_t *top_ids, float *top_logprobs,
                       void *stream) {
    const size_t b = float_bytes(dtype);
    if (!b || top_k > qvl::kMaxTopK) return QVL_ERR_UNSUPPORTED;
    if (n_rows == 0) return QVL_OK;
    if (!tokens || !logprobs || top_k < 0 || (top_k && (!top_ids || !top_logprobs))) return QVL_ERR_INVALID;
    if (vocab == 0 || vocab > (1u << 30) || n_rows > (1u << 27) || stride < vocab || stride > (size_t)INT32_MAX ||
        (size_t)top_k > vocab)
        return QVL_ERR_INVALID;
    if (!logits || ((uintptr_t)logits & (b - 1)) || !al4(tokens) || !al4(logprobs) || !al4(entropy) ||
        !al4(top_ids) || !al4(top_logprobs))
        return QVL_ERR_INVALID;
    const qvl::LogprobArgs a{logits, (long)stride, tokens, logprobs, entropy, top_ids, top_logprobs, (int)n_rows,
                             (int)vocab, top_k, dtype};
    QVL_CUDA_TRY(qvl::launch_token_logprobs(a, (cudaStream_t)stream));
    return QVL_OK;
}

// The same calls with their arguments as 64-bit words in the order of the
// declarations (floats as doubles), the stream last: a binding converts one
// buffer instead of three dozen arguments.
int qvl_internal_serving(int op, const int64_t *w) {
    auto p = [w](int i) { return reinterpret_cast<void *>(w[i]); };
    auto i32 = [w](int i) { return reinterpret_cast<int32_t *>(w[i]); };
    auto f32 = [w](int i) { return reinterpret_cast<float *>(w[i]); };
    auto z = [w](int i) { return (size_t)w[i]; };
    auto n = [w](int i) { return (int)w[i]; };
    auto real = [w](int i) {
        double d;
        memcpy(&d, &w[i], sizeof(d));
        return (float)d;
    };
    auto dims = [w](int i) { return reinterpret_cast<const qvl_attn_dims *>(w[i]); };
    switch (op) {
    case 0:
        return qvl_plan_pages(i32(0), i32(1), z(2), i32(3), n(4), n(5), i32(6), i32(7), z(8), i32(9), i32(10), i32(11),
                              i32(12), i32(13), i32(14), z(15), p(16));
    case 1:
        return qvl_qknorm_mrope_kv_append(p(0), p(1), p(2), n(3), z(4), z(5), z(6), p(7), p(8), p(9), n(10), z(11), i32(12),
                                          i32(13), z(14), n(15), i32(16), z(17), f32(18), f32(19), p(20), f32(21), p(22),
                                          f32(23), n(24), z(25), real(26), dims(27), p(28));
    case 2:
        return qvl_tree_attention(p(0), n(1), z(2), p(3), p(4), n(5), z(6), i32(7), i32(8), i32(9), i32(10), z(11), z(12),
                                  n(13), n(14), real(15), p(16), dims(17), p(18), z(19), p(20));
    case 3:
        return qvl_token_logprobs(p(0), n(1), z(2), i32(3), z(4), z(5), n(6), f32(7), f32(8), i32(9), f32(10), p(11));
    }
    return QVL_ERR_INVALID;
}

}  // extern "C"
