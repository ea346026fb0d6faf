// The forward of the selective scan for bf16 tensors.
#include "selective_scan_fwd.cuh"

namespace oxc {
template oxc_status selective_fwd_launch<bf16>(const SelectiveArgs<bf16>&, cudaStream_t);
}  // namespace oxc
