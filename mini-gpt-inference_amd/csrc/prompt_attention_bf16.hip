// prompt_attention_bf16.hip -- the kernels of prompt_attention.h for bf16 (a file per type, compiled side by side).
#include "prompt_attention.h"

namespace mgi {

hipError_t launch_prompt_bf16(const PromptArgs& a, hipStream_t stream) { return launch_prompt<bf16_t>(a, stream); }

}  // namespace mgi
