// Host side of the entry points of prompts' attention, of adapters and of the choice of experts: the argument checks.
#include "nvq_internal.h"

using namespace nvq;

static int32_t check_adapters(const nvq_adapters_desc *d) {
    const char *op = "apply_adapters";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    NVQ_TRY(check_float(op, d->dtype));
    if (d->rows < 0 || d->inputs < 0 || d->outputs < 0 || d->adapters < 0 || d->rank < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative size", op);
    if (d->x_stride < 0 || d->y_stride < 0 || d->out_stride < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative stride", op);
    if (d->rank > 256) return fail(NVQ_UNSUPPORTED, "%s: rank %d (256 at most)", op, d->rank);
    // (blocks of 16 rows and of 256 columns, and a share of the first product that 64 bits address)
    if (d->rows >= 1LL << 26 || d->outputs >= 1LL << 23 || d->inputs >= 1LL << 31 || d->adapters >= 1LL << 31)
        return fail(NVQ_UNSUPPORTED, "%s: 2^26 rows, 2^31 inputs, 2^23 outputs or 2^31 adapters", op);
    return NVQ_OK;
}

static int32_t check_prompt(const nvq_prompt_attention_desc *d) {
    const char *op = "prompt_attention";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    NVQ_TRY(check_float(op, d->dtype));
    if (d->rows < 0 || d->keys < 0 || d->query_heads < 0 || d->key_heads < 0 || d->sequences < 0 || d->window < 0 || d->head_dim < 0)
        return fail(NVQ_INVALID_ARGUMENT, "%s: negative size", op);
    if (d->key_heads == 0 || d->query_heads % d->key_heads != 0)
        return fail(NVQ_INVALID_ARGUMENT, "%s: %lld query heads over %lld key heads", op, (long long)d->query_heads, (long long)d->key_heads);
    if (d->window > 0 && !d->causal) return fail(NVQ_INVALID_ARGUMENT, "%s: a window without the causal mask", op);
    if (d->head_dim < 8 || d->head_dim > 256 || d->head_dim % 8 != 0) return fail(NVQ_UNSUPPORTED, "%s: heads of %d values (a multiple of 8 up to 256)", op, d->head_dim);
    if (d->query_heads >= 1 << 15 || d->rows >= 1LL << 30 || d->rows * d->query_heads >= 1LL << 30 || d->keys >= 1LL << 30 || d->sequences >= 1 << 20)
        return fail(NVQ_UNSUPPORTED, "%s: 2^30 rows and heads, 2^30 keys or 2^20 sequences", op);
    for (int i = 0; i < 2; i++)
        if (d->q_strides[i] < 0 || d->k_strides[i] < 0 || d->v_strides[i] < 0 || d->out_strides[i] < 0) return fail(NVQ_INVALID_ARGUMENT, "%s: negative stride", op);
    if (d->keys > 1 && (d->k_strides[0] >= 1 << 24 || d->v_strides[0] >= 1 << 24))  // (offsets within a tile are of 32 bits)
        return fail(NVQ_UNSUPPORTED, "%s: keys %lld and values %lld elements apart (less than 2^24)", op, (long long)d->k_strides[0], (long long)d->v_strides[0]);
    if (!prompt_attention_launchable(*d)) return fail(NVQ_UNSUPPORTED, "%s: %lld rows of %lld sequences, %lld heads each, in one launch", op, (long long)d->rows, (long long)d->sequences, (long long)d->query_heads);
    return NVQ_OK;
}

extern "C" {

size_t nvq_prompt_attention_workspace_bytes(const nvq_prompt_attention_desc *d) {
    if (check_prompt(d) != NVQ_OK || require_device() != NVQ_OK) return 0;
    return prompt_attention_workspace_bytes(*d);
}

int32_t nvq_prompt_attention(const nvq_prompt_attention_desc *d, const void *q, const void *k, const void *v, const int32_t *query_starts,
                             const int32_t *key_starts, const void *sinks, void *out, void *workspace, void *stream) {
    const char *op = "prompt_attention";
    NVQ_TRY(check_prompt(d));
    if (d->rows == 0 || d->query_heads == 0 || d->sequences == 0) return NVQ_OK;
    if (query_starts == nullptr && d->sequences != 1) return fail(NVQ_INVALID_ARGUMENT, "%s: %lld sequences without query starts", op, (long long)d->sequences);
    if (key_starts == nullptr && d->sequences != 1 && d->keys != d->rows)
        return fail(NVQ_INVALID_ARGUMENT, "%s: %lld rows and %lld keys of %lld sequences without key starts", op, (long long)d->rows, (long long)d->keys, (long long)d->sequences);
    if (q == nullptr || out == nullptr || (d->keys > 0 && (k == nullptr || v == nullptr))) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    for (const void *p : {q, k, v, sinks, (const void *)out}) NVQ_TRY(check_aligned(op, "an operand", p, (size_t)dtype_size(d->dtype)));
    NVQ_TRY(check_aligned(op, "workspace", workspace));
    NVQ_TRY(require_device());
    if (workspace == nullptr && prompt_attention_workspace_bytes(*d) != 0) return fail(NVQ_INVALID_ARGUMENT, "%s: null workspace", op);
    const PromptAttentionOperands o{q, k, v, sinks, query_starts, key_starts == nullptr && d->sequences != 1 ? query_starts : key_starts, out, workspace};
    return launch_prompt_attention(*d, o, (hipStream_t)stream);
}

size_t nvq_apply_adapters_workspace_bytes(const nvq_adapters_desc *d) {
    if (check_adapters(d) != NVQ_OK || require_device() != NVQ_OK || d->rows == 0) return 0;
    return adapters_workspace_bytes(*d);
}

int32_t nvq_apply_adapters(const nvq_adapters_desc *d, const void *x, const void *down, const void *up, const float *scales, const int32_t *ids,
                           const void *y, void *out, void *workspace, void *stream) {
    const char *op = "apply_adapters";
    NVQ_TRY(check_adapters(d));
    if (d->rows == 0 || d->outputs == 0) return NVQ_OK;
    if (ids == nullptr || y == nullptr || out == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    if (d->adapters > 0 && (d->inputs < 1 || d->rank < 1)) return fail(NVQ_INVALID_ARGUMENT, "%s: adapters of rank %d over %lld inputs", op, d->rank, (long long)d->inputs);
    if (d->adapters > 0 && (x == nullptr || down == nullptr || up == nullptr)) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    for (const void *p : {x, down, up, y, (const void *)out}) NVQ_TRY(check_aligned(op, "an operand", p, (size_t)dtype_size(d->dtype)));
    NVQ_TRY(check_aligned(op, "workspace", workspace));
    NVQ_TRY(require_device());
    if (workspace == nullptr && adapters_workspace_bytes(*d) != 0) return fail(NVQ_INVALID_ARGUMENT, "%s: null workspace", op);
    return launch_adapters(*d, x, down, up, scales, ids, y, out, workspace, (hipStream_t)stream);
}

int32_t nvq_moe_select(const nvq_moe_select_desc *d, const void *logits, const float *bias, int32_t *indices, void *weights, void *stream) {
    const char *op = "moe_select";
    if (d == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null descriptor", op);
    NVQ_TRY(check_float(op, d->dtype));
    if (d->scores != NVQ_SCORES_SOFTMAX && d->scores != NVQ_SCORES_SIGMOID) return fail(NVQ_INVALID_ARGUMENT, "%s: unknown scores %d", op, d->scores);
    if (d->rows < 0 || d->experts < 1) return fail(NVQ_INVALID_ARGUMENT, "%s: logits of shape [%lld, %d]", op, (long long)d->rows, d->experts);
    if (d->groups < 1 || d->experts % d->groups != 0 || d->top_groups < 1 || d->top_groups > d->groups)
        return fail(NVQ_INVALID_ARGUMENT, "%s: the best %d of %d groups of %d experts", op, d->top_groups, d->groups, d->experts);
    if (d->group_best != 1 && d->group_best != 2) return fail(NVQ_INVALID_ARGUMENT, "%s: a group's best %d (1 or 2)", op, d->group_best);
    const int32_t open = d->experts / d->groups * d->top_groups;
    if (d->k < 1 || d->k > open) return fail(NVQ_INVALID_ARGUMENT, "%s: k must be in 1..=%d, got %d", op, open, d->k);
    if (d->experts > 1024 || d->k > 64 || d->groups > 64)
        return fail(NVQ_UNSUPPORTED, "%s: %d experts in %d groups, k = %d: up to 1024, 64 and 64", op, d->experts, d->groups, d->k);
    if (d->rows >= 1LL << 26 || !launchable((d->rows + 3) / 4, 256)) return fail(NVQ_UNSUPPORTED, "%s: %lld rows (2^26 - 4 at most)", op, (long long)d->rows);
    if (d->rows == 0) return NVQ_OK;
    if (logits == nullptr || indices == nullptr || weights == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    for (const void *p : {logits, (const void *)weights}) NVQ_TRY(check_aligned(op, "an operand", p, (size_t)dtype_size(d->dtype)));
    NVQ_TRY(require_device());
    return launch_moe_select(*d, logits, bias, indices, weights, (hipStream_t)stream);
}

}  // extern "C"
