// paged_shared_f32.hip -- the kernels of paged_shared.h for f32 (a file per type, compiled side by side).
#include "paged_shared.h"

namespace mgi {

hipError_t launch_paged_shared_f32(const SharedArgs& a, hipStream_t stream) { return launch_type<float>(a, stream); }

}  // namespace mgi
