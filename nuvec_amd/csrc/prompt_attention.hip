// Attention of whole prompts: the sizes of its launches and workspace (prompt_kernel.h has the mathematics).
#include "prompt_attention.h"

namespace nvq {

namespace {

// Tiles of 32 keys of an item at least, where a block's keys are shared.  (bfloat16, 32 heads of 128 over 8 key heads: 61 rows over 512 keys 16.4 us, with eight
// tiles 18.8, not shared 18.9; 300 rows over 1000 keys 29.2, 28.8 with eight, 31.4 with sixteen; one row over 32768 keys 41 us, not shared 703.  In an
// earlier form a target of twice the blocks that the chip holds took 1.0, 1.25 and 1.4 times as long.)
constexpr int32_t kLeast = 4;

// Blocks that the chip holds.
int32_t target_of(const nvq_prompt_attention_desc &d) { return prompt::blocks_of((int)dtype_size(d.dtype), prompt::padded_dim(d.head_dim)) * compute_units(); }
// Units at most, whatever the starts on the device say: every sequence's last block of lines may be short.
int64_t most_units(const nvq_prompt_attention_desc &d) {
    const int64_t lines = d.rows * (d.query_heads / d.key_heads);
    return (lines / prompt::kLines + d.sequences) * d.key_heads;
}
// The device decides by the lengths, which are at most all keys.  One sequence of all rows is as the host sees it: its blocks of lines are split where
// they are fewer than the target.
bool may_split(const nvq_prompt_attention_desc &d, bool starts) {
    return d.keys > 2 * kScheduleKeys * kLeast && (starts || (d.rows * (d.query_heads / d.key_heads) + prompt::kLines - 1) / prompt::kLines * d.key_heads < target_of(d));
}
// Items of sequences that are split: at most twice the target (paged_schedule.h), and no more than their units have.
int64_t most_states(const nvq_prompt_attention_desc &d) {
    const int64_t splits = (d.keys + kScheduleKeys * kLeast - 1) / (kScheduleKeys * kLeast), all = most_units(d) * splits, full = 2 * (int64_t)target_of(d);
    return all < full ? all : full;
}

}  // namespace

bool prompt_attention_launchable(const nvq_prompt_attention_desc &d) { return launchable(most_units(d) + (1 << 12), 256); }

size_t prompt_attention_workspace_bytes(const nvq_prompt_attention_desc &d) {
    if (!may_split(d, true) || d.rows == 0) return 0;
    return prompt::kPlanBytes + (size_t)(most_states(d) * prompt::kLines * (prompt::padded_dim(d.head_dim) + 4)) * sizeof(float);
}

int32_t launch_prompt_attention(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, hipStream_t s) {
    const bool split = may_split(d, o.query_starts != nullptr || o.key_starts != nullptr);
    prompt::PromptLaunch r{};
    prompt::PromptBatch &b = r.batch;
    b.starts = o.query_starts, b.key_starts = o.key_starts, b.rows = d.rows, b.keys = d.keys;
    b.window = d.window < 1LL << 30 ? d.window : 1LL << 30;  // (as good as any larger one, and sums with it stay far from 64 bits)
    b.sequences = (int32_t)d.sequences, b.key_heads = (int32_t)d.key_heads, b.rep = (int32_t)(d.query_heads / d.key_heads), b.causal = d.causal != 0;
    b.few = -1, b.target = target_of(d), b.least = split ? kLeast : 1 << 26;
    const int64_t units = most_units(d), least = (int64_t)kScheduleKeys * kLeast, splits = split ? (d.keys + least - 1) / least : 1;
    const int64_t full = b.target, spare = full / 2 + units, items = full > spare ? full : spare;
    r.grid = (uint32_t)(units * splits < items ? units * splits : items);
    r.slots = split ? (int32_t)most_states(d) : 0;
    // (the last of the units that short sequences might have are seldom there)
    const int32_t cus = compute_units() & ~7;
    if (full > cus && units > cus && units <= full + cus / 4) r.turn = cus, r.back = (int32_t)(units < 2 * cus ? units : 2 * cus) - cus & ~7;
    r.merge_units = split ? (uint32_t)(units < full ? units : full) : 0;
    if (d.dtype == NVQ_F32) return prompt::launch_f32(d, o, r, s);
    return d.dtype == NVQ_BF16 ? prompt::launch_bf16(d, o, r, s) : prompt::launch_f16(d, o, r, s);
}

}  // namespace nvq
