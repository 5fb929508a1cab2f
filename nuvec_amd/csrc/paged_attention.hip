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
    b.lengths = o.lengths, b.starts = o.starts, b.rows = d.rows;
    b.window = d.window < 1LL << 30 ? d.window : 1LL << 30;  // (as good as any larger one, and sums with it stay far from 64 bits)
    b.sequences = (int32_t)c.sequences, b.key_heads = (int32_t)c.key_heads, b.rep = (int32_t)(d.query_heads / c.key_heads), b.causal = d.causal;
    b.few = INT32_MAX;
    return b;
}

}  // namespace paged

namespace {

// Lines of a sequence that the kernel of few lines takes, where the other kernel has the type: four units of it, two where they are of 16 lines.  (8
// sequences of 4096 positions, 4 heads of 128 on each of 8 key heads, 4 bits.  Groups of 64: 16 lines a sequence 31 us against the other's 40, 32 lines
// 43 against 42, 40 lines 53 against 43, 64 lines 60 against 44; of 32: 16 lines 39 against 46, 20 lines 61 against 49; of 128: 32 lines 34 against
// 36, 48 lines 40 against 37, 64 lines 47 against 39.  One sequence, groups of 64: 32 lines 17 against 19, 64 lines 22 against 20.)
int32_t few_lines(const nvq_paged_attention_desc &d) { return d.cache.head_dim / d.cache.group_size == 4 ? 16 : 32; }
constexpr int64_t kPromptLines = 128;

struct Kernel {
    int64_t lines;   // of a unit
    int32_t target;  // blocks that the chip holds at once
    size_t bytes;    // of its states
};
int64_t lines_of(const nvq_paged_attention_desc &d, bool many) { return many ? kPromptLines : 16 / (d.cache.head_dim / d.cache.group_size); }
// States of every item of the sequences that are split: at most twice the target (paged_schedule.h: each of their splits but the last is a
// whole item).
Kernel kernel_of(const nvq_paged_attention_desc &d, bool many) {
    const int groups = d.cache.head_dim / d.cache.group_size;
    Kernel k;
    k.lines = lines_of(d, many);
    k.target = (many || d.cache.dtype == NVQ_F32 || groups == 4 ? 2 : 3) * compute_units();
    k.bytes = paged::kPlanBytes + (size_t)(2 * (int64_t)k.target * k.lines * (d.cache.head_dim + 4)) * sizeof(float);
    return k;
}

// Tiles of an item at least, of few and of many lines.  (4 in place of 8 for many: one prompt of 20 rows over 300 positions 21 -> 16 us, three of 45 over
// 500 27 -> 24, one of 512 over as many 27.5 -> 29.4.)
constexpr int32_t kLeastFew = 8, kLeastMany = 4;
// (the device decides by the lengths, which are at most the table's columns; up to 8 tiles a second launch costs more than it saves)
bool may_split(const nvq_paged_attention_desc &d) { return d.cache.columns * d.cache.page_size > kScheduleKeys * kLeastFew; }
// Whether a sequence may have more lines than the kernel of few takes.
bool takes_many(const nvq_paged_attention_desc &d, bool starts) {
    const int64_t most = d.max_queries < d.rows ? d.max_queries : d.rows;
    return starts && d.cache.dtype != NVQ_F32 && most * (d.query_heads / d.cache.key_heads) > few_lines(d);
}

// Units of one of the kernels at most, whatever the lengths and starts on the device say.  `many`: whether both kernels are launched, or that of many
// lines alone.
int64_t most_units(const nvq_paged_attention_desc &d, bool starts, bool many, bool of_many) {
    const nvq_paged_desc &c = d.cache;
    const int64_t rep = d.query_heads / c.key_heads, lines = lines_of(d, of_many);
    const int64_t each = many && !of_many ? (few_lines(d) + lines - 1) / lines : (rep + lines - 1) / lines;
    int64_t units = c.sequences * each;
    if (starts) units = of_many ? d.rows * rep / lines + c.sequences : (d.rows * rep + lines - 1) / lines + c.sequences;
    if (many && !of_many && units > c.sequences * each) units = c.sequences * each;
    return units * c.key_heads;
}

}  // namespace

// (2^12 blocks: more than the items that splits add, half of what the chip holds)
bool paged_attention_launchable(const nvq_paged_attention_desc &d, bool starts) {
    const bool many = takes_many(d, starts);
    return launchable(most_units(d, starts, many, false) + (1 << 12), 256) && (!many || launchable(most_units(d, starts, many, true) + (1 << 12), 512));
}

size_t paged_attention_workspace_bytes(const nvq_paged_attention_desc &d) {
    if (!may_split(d) || d.rows == 0) return 0;
    return kernel_of(d, false).bytes + (takes_many(d, true) ? kernel_of(d, true).bytes : 0);
}

int32_t launch_paged_attention(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, hipStream_t s) {
    const nvq_paged_desc &c = d.cache;
    const bool starts = o.starts != nullptr, many = takes_many(d, starts), alone = many && c.sequences == 1;  // (alone: one launch, whatever its lines)
    auto launch_of = [&](bool of_many) {
        const Kernel k = kernel_of(d, of_many);
        paged::PagedLaunch r{};
        r.batch = paged::batch_of(d, o);
        r.batch.few = alone ? -1 : many ? few_lines(d) : INT32_MAX, r.batch.target = k.target;
        const int64_t rep = r.batch.rep, units = most_units(d, starts, many, of_many);  // (and so many items at most: paged_schedule.h)
        r.batch.least = !may_split(d) ? 1 << 26 : of_many ? kLeastMany : kLeastFew;
        const int64_t least = (int64_t)kScheduleKeys * r.batch.least, splits = (c.columns * c.page_size + least - 1) / least, full = k.target, spare = full / 2 + units;
        const int64_t items = full > spare ? full : spare;
        r.grid = (uint32_t)(units * splits < items ? units * splits : items);
        r.merge_units = may_split(d) ? (uint32_t)(units < full ? units : full) : 0;
        r.merge_lines = (uint32_t)(!starts && rep < k.lines ? rep : k.lines);
        r.states = of_many ? kernel_of(d, false).bytes : 0;
        return r;
    };
    paged::PagedLaunch few{};
    if (!alone) {
        few = launch_of(false), few.merged_later = many;
        const int32_t rc = c.dtype == NVQ_F32 ? paged::launch_rows_f32(d, o, few, s) : c.dtype == NVQ_BF16 ? paged::launch_rows_bf16(d, o, few, s) : paged::launch_rows_f16(d, o, few, s);
        if (rc != NVQ_OK || !many) return rc;
    }
    return c.dtype == NVQ_BF16 ? paged::launch_prompt_bf16(d, o, few, launch_of(true), s) : paged::launch_prompt_f16(d, o, few, launch_of(true), s);
}

}  // namespace nvq
