// Attention over a paged, affine-quantized cache: the choice of kernels and their launches (paged_rows_kernel.h has the mathematics).
#include "paged_attention.h"

#include "paged_rows_kernel.h"

namespace nvq {
namespace paged {

PagedBatch batch_of(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o) {
    const nvq_paged_desc &c = d.cache;
    PagedBatch b{};
    b.place.table = o.page_table, b.place.stride = c.table_stride, b.place.pages = c.pages;
    b.place.sequences = (int32_t)c.sequences, b.place.columns = (int32_t)c.columns;
    while ((1LL << b.place.page_shift) < c.page_size) b.place.page_shift++;
    b.lengths = o.lengths, b.starts = o.starts, b.rows = d.rows, b.window = d.window;
    b.sequences = (int32_t)c.sequences, b.key_heads = (int32_t)c.key_heads, b.rep = (int32_t)(d.query_heads / c.key_heads), b.causal = d.causal;
    b.few = INT32_MAX;
    return b;
}

}  // namespace paged

namespace {

// Blocks of the kernel of few lines that the chip holds at once.
int32_t rows_target(const nvq_paged_attention_desc &d) {
    return (d.cache.dtype == NVQ_F32 || d.cache.head_dim / d.cache.group_size == 4 ? 2 : 3) * compute_units();
}

// (the device decides by the lengths, which are at most the table's columns)
bool may_split(const nvq_paged_attention_desc &d) { return d.cache.columns * d.cache.page_size > 32 * 8; }

}  // namespace

// States of every item of the sequences that are split: at most twice the target (paged_schedule.h: each of their splits but the last
// is a whole item).
size_t paged_attention_workspace_bytes(const nvq_paged_attention_desc &d) {
    if (!may_split(d) || d.rows == 0) return 0;
    const int64_t lines = 16 / (d.cache.head_dim / d.cache.group_size);
    return (size_t)(2 * (int64_t)rows_target(d) * lines * (d.cache.head_dim + 2)) * sizeof(float);
}

int32_t launch_paged_attention(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, hipStream_t s) {
    paged::RowsLaunch r{};
    const nvq_paged_desc &c = d.cache;
    r.batch = paged::batch_of(d, o);
    r.batch.target = rows_target(d);
    const int64_t lines = 16 / (c.head_dim / c.group_size), rep = r.batch.rep;
    // At most so many units and items, whatever the lengths and starts on the device say (paged_schedule.h).
    const int64_t most = c.key_heads * (o.starts == nullptr ? c.sequences * ((rep + lines - 1) / lines) : (d.rows * rep + lines - 1) / lines + c.sequences);
    const int64_t splits = (c.columns * c.page_size + 255) / 256, full = r.batch.target, spare = full / 2 + most;
    const int64_t items = full > spare ? full : spare;
    r.grid = (uint32_t)(most * splits < items ? most * splits : items);
    r.merge_units = may_split(d) ? (uint32_t)(most < full ? most : full) : 0;
    r.merge_lines = (uint32_t)(o.starts == nullptr && rep < lines ? rep : lines);
    switch (c.dtype) {
    case NVQ_F32: return paged::launch_rows_f32(d, o, r, s);
    case NVQ_BF16: return paged::launch_rows_bf16(d, o, r, s);
    default: return paged::launch_rows_f16(d, o, r, s);
    }
}

}  // namespace nvq
