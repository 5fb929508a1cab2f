// Host side of the heads' and the paged cache's entry points: the argument checks.
#include "nvq_internal.h"

namespace nvq {
namespace {

int32_t check_rotation(const char *op, int32_t head_dim, int32_t rotary_dims, int64_t table_rows, const void *table) {
    if (rotary_dims < 0 || rotary_dims > head_dim || rotary_dims % 2 != 0)
        return fail(NVQ_INVALID_ARGUMENT, "%s: %d rotary values of heads of %d", op, rotary_dims, head_dim);
    if (rotary_dims > 0 && (table_rows < 1 || table == nullptr)) return fail(NVQ_INVALID_ARGUMENT, "%s: no table of angles", op);
    return check_aligned(op, "the table of angles", table, 8);
}

int32_t check_elements(const char *op, const char *what, const void *p, int32_t dtype) { return check_aligned(op, what, p, (size_t)dtype_size(dtype)); }

int32_t check_eps(const char *op, double eps) {
    return eps >= 0.0 && eps < 1e30 ? NVQ_OK : fail(NVQ_INVALID_ARGUMENT, "%s: eps %g", op, eps);
}

int32_t check_paged(const char *op, const nvq_paged_desc &c) {
    NVQ_TRY(check_float(op, c.dtype));
    const nvq_quant quant{NVQ_AFFINE, c.group_size, c.bits};
    NVQ_TRY(check_quant(&quant, op));
    if (c.pages < 0 || c.page_size < 0 || c.key_heads < 0 || c.sequences < 0 || c.columns < 0 || c.head_dim < 0)
        return fail(NVQ_INVALID_ARGUMENT, "%s: negative size", op);
    if ((c.head_dim != 64 && c.head_dim != 128) || (c.bits != 4 && c.bits != 8) || c.head_dim % c.group_size != 0)
        return fail(NVQ_UNSUPPORTED, "%s: paged caches have heads of 64 or 128 values in 4 or 8 bits, in whole groups", op);
    if (c.page_size < 16 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)) != 0)
        return fail(NVQ_UNSUPPORTED, "%s: pages of %lld positions (a power of two from 16 to 1024)", op, (long long)c.page_size);
    if (c.sequences > 1 && c.table_stride < c.columns) return fail(NVQ_INVALID_ARGUMENT, "%s: the page table's rows overlap", op);
    if (c.pages >= 1LL << 31 || c.key_heads >= 1 << 15 || c.sequences >= 1 << 20 || c.columns > ((1LL << 30) - 1) / c.page_size)
        return fail(NVQ_UNSUPPORTED, "%s: more than 2^31 pages, 2^15 key heads, 2^20 sequences or 2^30 positions of one", op);
    return NVQ_OK;
}

// The page of every token is looked up before anything else of the pool, which may be empty.
int32_t check_page_table(const char *op, const nvq_paged_desc &c, const int32_t *page_table) {
    return c.sequences > 0 && c.columns > 0 && page_table == nullptr ? fail(NVQ_INVALID_ARGUMENT, "%s: null page table", op) : NVQ_OK;
}

int32_t check_pool(const char *op, const nvq_paged_desc &c, const void *kw, const void *ks, const void *kb, const void *vw, const void *vs,
                   const void *vb) {
    if (kw == nullptr || ks == nullptr || kb == nullptr || vw == nullptr || vs == nullptr || vb == nullptr)
        return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    NVQ_TRY(check_aligned(op, "keys", kw));
    NVQ_TRY(check_aligned(op, "values", vw));
    for (const void *p : {ks, kb, vs, vb}) NVQ_TRY(check_elements(op, "scales and biases", p, c.dtype));
    return NVQ_OK;
}

}  // namespace
}  // namespace nvq

using namespace nvq;

template <typename F>
static int32_t rotation_table(const F *freqs, int32_t dims, int64_t rows, double base, double scale, double magnitude, float *table, void *stream) {
    const char *op = "rotation_table";
    if (dims < 0 || dims % 2 != 0 || rows < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: %d values, %lld positions", op, dims, (long long)rows);
    if (dims == 0 || rows == 0) return NVQ_OK;
    if (rows >= (1LL << 32) || !launchable((rows * (dims / 2) + 255) / 256, 256)) return fail(NVQ_UNSUPPORTED, "%s: 2^32 angles or more", op);
    if (freqs == nullptr && !(base > 0.0)) return fail(NVQ_INVALID_ARGUMENT, "%s: base %g", op, base);
    if (table == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    NVQ_TRY(require_device());
    NVQ_TRY(check_aligned(op, "the table of angles", table, 8));
    NVQ_TRY(check_aligned(op, "the frequencies", freqs, sizeof(F)));
    return launch_rotation_table(freqs, dims / 2, rows, base, scale, magnitude, table, (hipStream_t)stream);
}

extern "C" {

int32_t nvq_rotation_table(const float *freqs, int32_t dims, int64_t rows, double base, double scale, double magnitude, float *table, void *stream) {
    return rotation_table(freqs, dims, rows, base, scale, magnitude, table, stream);
}

int32_t nvq_rotation_table_f64(const double *freqs, int32_t dims, int64_t rows, double base, double scale, double magnitude, float *table, void *stream) {
    return rotation_table(freqs, dims, rows, base, scale, magnitude, table, stream);
}

int32_t nvq_head_norm_rope(const nvq_head_rope_desc *d, const float *table, const int32_t *offsets, const void *x0, const void *weight0, void *y0,
                           const void *x1, const void *weight1, void *y1, void *stream) {
    const char *op = "head_norm_rope";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    NVQ_TRY(check_float(op, d->dtype));
    if (d->head_dim < 1 || d->batch < 0 || d->length < 0 || d->heads[0] < 0 || d->heads[1] < 0)
        return fail(NVQ_INVALID_ARGUMENT, "%s: negative size, or heads of no values", op);
    if (d->head_dim > 512) return fail(NVQ_UNSUPPORTED, "%s: heads of %d values (512 at most)", op, d->head_dim);
    NVQ_TRY(check_rotation(op, d->head_dim, d->rotary_dims, d->table_rows, table));
    NVQ_TRY(check_eps(op, d->eps));
    // (a row of blocks a head where there are few positions)
    const int64_t most = most_positions(d->head_dim);
    if (d->heads[0] >= 1 << 16 || d->heads[1] >= 1 << 16 || d->heads[0] + d->heads[1] >= 1 << 16 || (d->length > 0 && d->batch > most / d->length))
        return fail(NVQ_UNSUPPORTED, "%s: more than 2^16 heads or %lld positions of %d values", op, (long long)most, d->head_dim);
    if (d->batch == 0 || d->length == 0 || d->heads[0] + d->heads[1] == 0) return NVQ_OK;
    const void *const x[2] = {x0, x1}, *const w[2] = {weight0, weight1};
    void *const y[2] = {y0, y1};
    for (int i = 0; i < 2; i++) {
        if (d->heads[i] == 0) continue;
        if (x[i] == nullptr || y[i] == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
        NVQ_TRY(check_elements(op, "an operand", x[i], d->dtype));
        NVQ_TRY(check_elements(op, "a weight", w[i], d->dtype));
        NVQ_TRY(check_elements(op, "an output", y[i], d->dtype));
    }
    NVQ_TRY(require_device());
    return launch_head_rope(*d, table, offsets, x, w, y, (hipStream_t)stream);
}

int32_t nvq_append_paged(const nvq_paged_append_desc *d, const int32_t *page_table, const int32_t *sequences, const int32_t *positions,
                         const float *table, const void *q, const void *q_weight, void *q_out, const void *k, const void *k_weight, const void *v,
                         uint32_t *k_w, void *k_s, void *k_b, uint32_t *v_w, void *v_s, void *v_b, void *stream) {
    const char *op = "append_paged";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    const nvq_paged_desc &c = d->cache;
    NVQ_TRY(check_paged(op, c));
    NVQ_TRY(check_rotation(op, c.head_dim, d->rotary_dims, d->table_rows, table));
    NVQ_TRY(check_eps(op, d->eps));
    if (d->tokens < 0 || d->query_heads < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative size", op);
    const int64_t most = most_positions(c.head_dim);
    if (d->tokens > most || d->query_heads >= 1 << 16 || d->query_heads + 2 * c.key_heads >= 1 << 16)  // (a row of blocks a head where there are few tokens)
        return fail(NVQ_UNSUPPORTED, "%s: more than %lld tokens or 2^16 heads of them", op, (long long)most);
    const bool queries = q != nullptr && d->query_heads > 0;
    if (d->tokens == 0 || (c.key_heads == 0 && !queries)) return NVQ_OK;
    if (positions == nullptr || (c.key_heads > 0 && (k == nullptr || v == nullptr)) || (queries && q_out == nullptr))
        return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    NVQ_TRY(check_page_table(op, c, page_table));
    if (c.key_heads > 0 && c.pages > 0 && c.sequences > 0 && c.columns > 0) NVQ_TRY(check_pool(op, c, k_w, k_s, k_b, v_w, v_s, v_b));
    for (const void *p : {q, q_weight, k, k_weight, v}) NVQ_TRY(check_elements(op, "an operand", p, c.dtype));
    NVQ_TRY(check_aligned(op, "the queries' output", q_out));
    NVQ_TRY(require_device());
    const PagedAppendOperands o{page_table, sequences, positions, table, queries ? q : nullptr, q_weight, k, k_weight, v, q_out, k_w, k_s, k_b, v_w, v_s, v_b};
    return launch_append_paged(*d, o, (hipStream_t)stream);
}

int32_t nvq_read_paged(const nvq_paged_desc *d, int64_t tokens, const int32_t *page_table, const int32_t *sequences, const int32_t *positions,
                       const uint32_t *k_w, const void *k_s, const void *k_b, const uint32_t *v_w, const void *v_s, const void *v_b, void *keys,
                       void *values, void *stream) {
    const char *op = "read_paged";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    NVQ_TRY(check_paged(op, *d));
    if (tokens < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative size", op);
    const int64_t most = most_positions(d->head_dim);
    if (tokens > most) return fail(NVQ_UNSUPPORTED, "%s: more than %lld tokens", op, (long long)most);
    if (tokens == 0 || d->key_heads == 0) return NVQ_OK;
    if (positions == nullptr || keys == nullptr || values == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    NVQ_TRY(check_page_table(op, *d, page_table));
    if (d->pages > 0 && d->sequences > 0 && d->columns > 0) NVQ_TRY(check_pool(op, *d, k_w, k_s, k_b, v_w, v_s, v_b));
    NVQ_TRY(check_aligned(op, "the keys' output", keys));
    NVQ_TRY(check_aligned(op, "the values' output", values));
    NVQ_TRY(require_device());
    PagedAppendOperands o{};
    o.page_table = page_table, o.sequences = sequences, o.positions = positions;
    o.kw = (void *)k_w, o.ks = (void *)k_s, o.kb = (void *)k_b, o.vw = (void *)v_w, o.vs = (void *)v_s, o.vb = (void *)v_b;
    return launch_read_paged(*d, tokens, o, keys, values, (hipStream_t)stream);
}

static int32_t check_paged_attention(const nvq_paged_attention_desc *d) {
    const char *op = "paged_attention";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    const nvq_paged_desc &c = d->cache;
    NVQ_TRY(check_paged(op, c));
    if (d->rows < 0 || d->query_heads < 0 || d->window < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative size", op);
    if (c.key_heads == 0 || d->query_heads % c.key_heads != 0)
        return fail(NVQ_INVALID_ARGUMENT, "%s: %lld query heads over %lld key heads", op, (long long)d->query_heads, (long long)c.key_heads);
    if (d->window > 0 && !d->causal) return fail(NVQ_INVALID_ARGUMENT, "%s: a window without the causal mask", op);
    if (d->query_heads >= 1 << 15 || d->rows >= 1LL << 30 || d->rows * d->query_heads >= 1LL << 30) return fail(NVQ_UNSUPPORTED, "%s: more than 2^30 rows and heads", op);
    for (int i = 0; i < 2; i++)
        if (d->q_strides[i] < 0 || d->out_strides[i] < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative stride", op);
    return NVQ_OK;
}

size_t nvq_paged_attention_workspace_bytes(const nvq_paged_attention_desc *d) {
    if (check_paged_attention(d) != NVQ_OK || require_device() != NVQ_OK) return 0;
    return paged_attention_workspace_bytes(*d);
}

int32_t nvq_paged_attention(const nvq_paged_attention_desc *d, const void *q, const uint32_t *k_w, const void *k_s, const void *k_b,
                            const uint32_t *v_w, const void *v_s, const void *v_b, const int32_t *page_table, const int32_t *lengths,
                            const int32_t *query_starts, const void *sinks, void *out, void *workspace, void *stream) {
    const char *op = "paged_attention";
    NVQ_TRY(check_paged_attention(d));
    const nvq_paged_desc &c = d->cache;
    if (d->rows == 0 || d->query_heads == 0 || c.sequences == 0) return NVQ_OK;
    if (query_starts == nullptr && c.sequences != d->rows)
        return fail(NVQ_INVALID_ARGUMENT, "%s: %lld rows of %lld sequences without query starts", op, (long long)d->rows, (long long)c.sequences);
    if (c.pages == 0 || c.columns == 0) return fail(NVQ_INVALID_ARGUMENT, "%s: a cache of no pages", op);
    if (!paged_attention_launchable(*d, query_starts != nullptr))
        return fail(NVQ_UNSUPPORTED, "%s: %lld rows of %lld sequences, %lld heads each, in one launch", op, (long long)d->rows, (long long)c.sequences, (long long)d->query_heads);
    if (q == nullptr || page_table == nullptr || lengths == nullptr || out == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    NVQ_TRY(check_pool(op, c, k_w, k_s, k_b, v_w, v_s, v_b));
    for (const void *p : {q, sinks, (const void *)out}) NVQ_TRY(check_elements(op, "an operand", p, c.dtype));
    NVQ_TRY(check_aligned(op, "workspace", workspace));
    NVQ_TRY(require_device());
    if (workspace == nullptr && paged_attention_workspace_bytes(*d) != 0) return fail(NVQ_INVALID_ARGUMENT, "%s: null workspace", op);
    const PagedAttentionOperands o{q, k_w, k_s, k_b, v_w, v_s, v_b, sinks, page_table, lengths, query_starts, out, workspace};
    return launch_paged_attention(*d, o, (hipStream_t)stream);
}

}  // extern "C"
