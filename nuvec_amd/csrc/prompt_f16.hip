// Attention of whole prompts, float16 (prompt_kernel.h).
#include "prompt_kernel.h"

namespace nvq {
namespace prompt {

int32_t launch_f16(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s) { return launch_type<f16_t>(d, o, r, s); }

}  // namespace prompt
}  // namespace nvq
