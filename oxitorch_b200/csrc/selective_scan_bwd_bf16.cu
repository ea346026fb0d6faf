// The VJP of the selective scan for bf16 tensors.
#include "selective_scan_bwd.cuh"

namespace oxc {
template oxc_status selective_bwd_launch<bf16>(const SelectiveArgs<bf16>&, float*, bf16*, bf16*, cudaStream_t);
}  // namespace oxc
