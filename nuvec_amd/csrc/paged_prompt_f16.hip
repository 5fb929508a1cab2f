// Attention of many lines over a paged cache, float16.
#include "paged_prompt_kernel.h"

namespace nvq {
namespace paged {

int32_t launch_prompt_f16(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &few, const PagedLaunch &r, hipStream_t s) {
    return launch_prompt<f16_t>(d, o, few, r, s);
}

}  // namespace paged
}  // namespace nvq
