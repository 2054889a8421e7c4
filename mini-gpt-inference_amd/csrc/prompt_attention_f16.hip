// prompt_attention_f16.hip -- the kernels of prompt_attention.h for f16 (a file per type, compiled side by side).
#include "prompt_attention.h"

namespace mgi {

hipError_t launch_prompt_f16(const PromptArgs& a, hipStream_t stream) { return launch_prompt<f16_t>(a, stream); }

}  // namespace mgi
