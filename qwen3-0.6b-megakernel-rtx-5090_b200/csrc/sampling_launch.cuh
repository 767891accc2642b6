// Launch of the sampling kernel: sampling_<type>_sm100.cu hold an instance each, so that they compile side by side.
#ifndef QMK_SAMPLING_LAUNCH_CUH_
#define QMK_SAMPLING_LAUNCH_CUH_

#include <algorithm>
#include <atomic>

#include "sampling.cuh"

namespace qmk_sample {

constexpr int DEVICES = 16;

template <typename T, int AN_SM>
struct Launch {
  static constexpr int SMEM = sizeof(Shared) + 2 * TURN * THREADS * 4 * sizeof(T);
  static void configure(cudaLaunchConfig_t *cfg, cudaLaunchAttribute *attr, int rows, int ranks, cudaStream_t stream) {
    *cfg = {};
    cfg->gridDim = dim3(static_cast<unsigned int>(rows) * ranks);
    cfg->blockDim = dim3(THREADS);
    cfg->dynamicSmemBytes = SMEM;
    cfg->stream = stream;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = ranks;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
  }
  // Rows whose clusters of `ranks` CTAs are resident together on this device; asked for once.  (Clusters lie inside a GPC, of which not all have as
  // many SMs: 16 clusters of eight CTAs on 128 of 148 SMs took two waves, 24 us where four CTAs a row took 17.)
  static cudaError_t resident(int device, int ranks, int *rows) {
    static std::atomic<int> known[DEVICES][4];
    std::atomic<int> &at = known[device][ranks == 8 ? 3 : ranks >> 1];
    if ((*rows = at.load()) > 0) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(sample_rows<T, AN_SM>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    configure(&cfg, &attr, 1, ranks, nullptr);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(rows, sample_rows<T, AN_SM>, &cfg);
    if (e == cudaSuccess) at.store(*rows = std::max(*rows, 1));
    return e;
  }
  static cudaError_t run(const Params &p, int rows, int ranks, cudaStream_t stream) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    configure(&cfg, &attr, rows, ranks, stream);
    return cudaLaunchKernelEx(&cfg, sample_rows<T, AN_SM>, p);
  }
};

// CTAs per row: as many as leave all rows resident at once, with at least 1024 tokens each; alone on their SMs where that is enough.
template <typename T>
cudaError_t launch_rows(const Params &p, int rows, cudaStream_t stream) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && device >= DEVICES) e = cudaErrorInvalidDevice;
  for (int ranks = MAX_CLUSTER; e == cudaSuccess; ranks /= 2) {
    if (ranks > 1 && p.vocab <= ranks / 2 * 1024) continue;
    int alone = 0, two = 0;
    e = Launch<T, 1>::resident(device, ranks, &alone);
    if (e == cudaSuccess && rows <= alone) return Launch<T, 1>::run(p, rows, ranks, stream);
    if (e == cudaSuccess) e = Launch<T, 2>::resident(device, ranks, &two);
    if (e == cudaSuccess && (rows <= two || ranks == 1)) return Launch<T, 2>::run(p, rows, ranks, stream);
  }
  return e;
}

}  // namespace qmk_sample
#endif  // QMK_SAMPLING_LAUNCH_CUH_
