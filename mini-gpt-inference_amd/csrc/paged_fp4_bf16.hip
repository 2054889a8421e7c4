// paged_fp4_bf16.hip -- the 4-bit pool's decode attention for bf16 queries.
#include "paged_fp4.h"

namespace mgi {

hipError_t launch_paged_fp4_bf16(const Fp4DecodeArgs& a, hipStream_t stream) { return launch_paged_fp4<bf16_t>(a, stream); }

}  // namespace mgi
