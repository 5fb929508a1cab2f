// Attention of whole prompts, float32 (prompt_kernel.h).
#include "prompt_kernel.h"

namespace nvq {
namespace prompt {

int32_t launch_f32(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s) { return launch_type<float>(d, o, r, s); }

}  // namespace prompt
}  // namespace nvq
