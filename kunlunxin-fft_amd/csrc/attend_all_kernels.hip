// attend_all_kernels.hip -- attention over the paged 8-bit cache: the
// kernels over what each sequence's queries see
// (attend_device.hpp).
#include "attend_device.hpp"

namespace mfft {

template void launch_part<kAll>(const mfft_cache&, const mfft_attend_args&, const AttendLaunch&, hipStream_t);

}  // namespace mfft
