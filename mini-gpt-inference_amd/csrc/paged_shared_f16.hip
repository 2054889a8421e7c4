// paged_shared_f16.hip -- the kernels of paged_shared.h for f16 (a file per type, compiled side by side).
#include "paged_shared.h"

namespace mgi {

hipError_t launch_paged_shared_f16(const SharedArgs& a, hipStream_t stream) { return launch_type<f16_t>(a, stream); }

}  // namespace mgi
