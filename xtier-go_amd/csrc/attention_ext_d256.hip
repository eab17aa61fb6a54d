// The kernels of attention_ext_kernels.hpp for heads of 256 dims.
#include "attention_ext_kernels.hpp"

namespace xtg::hip {

template void ext_launch<256>(const ExtCall&, const ExtPlan&, const ExtArgs&, int, hipStream_t, const Timed&);

}  // namespace xtg::hip
