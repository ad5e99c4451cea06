// attend_sinks_kernels.hip -- attention over the paged 8-bit cache: the
// kernels over the keys in a window and the first tokens, which stay visible
// (attend_device.hpp).
#include "attend_device.hpp"

namespace mfft {

template void launch_part<kSinks>(const mfft_cache&, const mfft_attend_args&, const AttendLaunch&, hipStream_t);

}  // namespace mfft
