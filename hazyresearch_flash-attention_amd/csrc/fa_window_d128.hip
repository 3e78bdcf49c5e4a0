// fa_window_d128.hip — the windowed and paged kernels of head_dim tile 128.
#include "fa_window_kernels_impl.h"

namespace fa {
template hipError_t launch_window_fwd<128>(const WinFwdArgs &, int, bool, WinShape, hipStream_t);
template hipError_t launch_window_bwd<128>(const WinBwdArgs &, int, const WinBwdPlan &, hipStream_t);
}  // namespace fa
