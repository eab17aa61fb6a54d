// The kernels of paged_attention_kernels.hpp for heads of 256 dims.
#include "paged_attention_kernels.hpp"

namespace xtg::hip {

template void paged_launch<256>(const PagedAttnCall&, const PagedPlan&, const PagedArgs&, hipStream_t, const PagedTimed&);

}  // namespace xtg::hip
