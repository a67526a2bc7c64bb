// The paged attention kernels over 8-bit pages.
#include "attn_paged_body.hpp"

namespace pelica {

hipError_t launch_paged_q8(const PagedParams& p, hipStream_t st) { return launch_paged_as<true>(p, st); }

}  // namespace pelica
