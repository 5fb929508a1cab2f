// The launches of attention over a paged cache, one translation unit per element type.
#pragma once

#include "nvq_internal.h"
#include "paged_schedule.h"

namespace nvq {
namespace paged {

struct RowsLaunch {
    PagedBatch batch;
    uint32_t grid, merge_units, merge_lines;  // merge_units 0: no sequence can be split
};
int32_t launch_rows_f32(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const RowsLaunch &r, hipStream_t s);
int32_t launch_rows_bf16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const RowsLaunch &r, hipStream_t s);
int32_t launch_rows_f16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const RowsLaunch &r, hipStream_t s);

}  // namespace paged
}  // namespace nvq
