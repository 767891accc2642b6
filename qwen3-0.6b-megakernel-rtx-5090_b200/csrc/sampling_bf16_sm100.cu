// sample_rows for bf16 logits.
#include "sampling_launch.cuh"

namespace qmk_sample {
cudaError_t launch_bf16(const Params &p, int rows, cudaStream_t stream) { return launch_rows<__nv_bfloat16>(p, rows, stream); }
}  // namespace qmk_sample
