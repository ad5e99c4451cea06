// attend_prefix_kernels.hip -- attention over the paged 8-bit cache: the
// kernels over the keys that groups of sequences share
// (attend_device.hpp).
#include "attend_device.hpp"

namespace mfft {

template void launch_part<kPrefix>(const mfft_cache&, const mfft_attend_args&, const AttendLaunch&, hipStream_t);

}  // namespace mfft
