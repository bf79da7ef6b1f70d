// The gated linear recurrence's kernels in f32 storage, in a translation unit of their own so that
// they compile in parallel.
#define HSN_SCAN_INSTANTIATE
#include "scan.cuh"

namespace hsn {
namespace scan {
template void launch_forward<float>(const Args&, int, bool, hipStream_t);
template void launch_backward<float>(const Args&, int, bool, hipStream_t);
}  // namespace scan
}  // namespace hsn
