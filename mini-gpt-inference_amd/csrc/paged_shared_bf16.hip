// paged_shared_bf16.hip -- the kernels of paged_shared.h for bf16 (a file per type, compiled side by side).
#include "paged_shared.h"

namespace mgi {

hipError_t launch_paged_shared_bf16(const SharedArgs& a, hipStream_t stream) { return launch_type<bf16_t>(a, stream); }

}  // namespace mgi
