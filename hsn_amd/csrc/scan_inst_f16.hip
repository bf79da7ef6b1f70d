// The gated linear recurrence's kernels in f16 storage, in a translation unit of their own so that
// they compile in parallel.
#define HSN_SCAN_INSTANTIATE
#include "scan.cuh"

namespace hsn {
namespace scan {
template void launch_forward<_Float16>(const Args&, int, bool, hipStream_t);
template void launch_backward<_Float16>(const Args&, int, bool, hipStream_t);
}  // namespace scan
}  // namespace hsn
