// paged_fp4_f32.hip -- the 4-bit pool's decode attention for f32 queries.
#include "paged_fp4.h"

namespace mgi {

hipError_t launch_paged_fp4_f32(const Fp4DecodeArgs& a, hipStream_t stream) { return launch_paged_fp4<float>(a, stream); }

}  // namespace mgi
