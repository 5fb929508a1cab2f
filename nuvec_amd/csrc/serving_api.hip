// Host side of the entry points of adapters and of the choice of experts: the argument checks.
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

extern "C" {

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
    if (d->rows >= 1LL << 26) return fail(NVQ_UNSUPPORTED, "%s: %lld rows (fewer than 2^26)", op, (long long)d->rows);
    if (d->rows == 0) return NVQ_OK;
    if (logits == nullptr || indices == nullptr || weights == nullptr) return fail(NVQ_INVALID_ARGUMENT, "%s: null operand", op);
    for (const void *p : {logits, (const void *)weights}) NVQ_TRY(check_aligned(op, "an operand", p, (size_t)dtype_size(d->dtype)));
    NVQ_TRY(require_device());
    return launch_moe_select(*d, logits, bias, indices, weights, (hipStream_t)stream);
}

}  // extern "C"
