// prompt_attention_f32.hip -- the kernels of prompt_attention.h for f32 (a file per type, compiled side by side).
#include "prompt_attention.h"

namespace mgi {

hipError_t launch_prompt_f32(const PromptArgs& a, hipStream_t stream) { return launch_prompt<float>(a, stream); }

}  // namespace mgi
