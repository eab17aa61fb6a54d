// The kernels of attention_ext_kernels.hpp for heads of 128 dims.
#include "attention_ext_kernels.hpp"

namespace xtg::hip {

template void ext_launch<128>(const ExtCall&, const ExtPlan&, const ExtArgs&, int, hipStream_t, const Timed&);

}  // namespace xtg::hip
