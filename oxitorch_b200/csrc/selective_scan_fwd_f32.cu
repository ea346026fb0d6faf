// The forward of the selective scan for f32 tensors.
#include "selective_scan_fwd.cuh"

namespace oxc {
template oxc_status selective_fwd_launch<float>(const SelectiveArgs<float>&, cudaStream_t);
}  // namespace oxc
