// sample_rows for fp32 logits.
#include "sampling_launch.cuh"

namespace qmk_sample {
cudaError_t launch_fp32(const Params &p, int rows, cudaStream_t stream) { return launch_rows<float>(p, rows, stream); }
}  // namespace qmk_sample
