// The launches of attention over a paged cache, one translation unit per element type and kernel.
#pragma once

#include "nvq_internal.h"
#include "paged_schedule.h"

namespace nvq {
namespace paged {

constexpr size_t kPlanBytes = 64;  // in front of a kernel's states

struct PagedLaunch {
    PagedBatch batch;
    size_t states;                            // where in the workspace the kernel's plan and states lie
    uint32_t grid, merge_units, merge_lines;  // merge_units 0: no sequence can be split
    bool merged_later;                        // the other kernel's merge takes these units too
};
// few lines: query rows x query heads of a key head
int32_t launch_rows_f32(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &r, hipStream_t s);
int32_t launch_rows_bf16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &r, hipStream_t s);
int32_t launch_rows_f16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &r, hipStream_t s);
// many; `few`: the launch of few lines in front of it, whose splits it merges with its own (grid 0: none)
int32_t launch_prompt_bf16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &few, const PagedLaunch &r, hipStream_t s);
int32_t launch_prompt_f16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &few, const PagedLaunch &r, hipStream_t s);

}  // namespace paged
}  // namespace nvq
