// Attention of whole prompts, bfloat16 (prompt_kernel.h).
#include "prompt_kernel.h"

namespace nvq {
namespace prompt {

int32_t launch_bf16(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s) { return launch_type<bf16_t>(d, o, r, s); }

}  // namespace prompt
}  // namespace nvq
