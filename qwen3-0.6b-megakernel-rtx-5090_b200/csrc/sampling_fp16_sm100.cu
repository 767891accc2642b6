// sample_rows for fp16 logits.
#include "sampling_launch.cuh"

namespace qmk_sample {
cudaError_t launch_fp16(const Params &p, int rows, cudaStream_t stream) { return launch_rows<__half>(p, rows, stream); }
}  // namespace qmk_sample
