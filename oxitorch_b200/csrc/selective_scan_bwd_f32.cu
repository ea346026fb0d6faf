// The VJP of the selective scan for f32 tensors.
#include "selective_scan_bwd.cuh"

namespace oxc {
template oxc_status selective_bwd_launch<float>(const SelectiveArgs<float>&, float*, float*, float*, cudaStream_t);
}  // namespace oxc
