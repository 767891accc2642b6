// C entry of the sampling kernel (sampling.cuh).
#include "../../include/qwen_megakernel.h"

#include <algorithm>
#include <atomic>
#include <string>

#include "engine_internal.h"
#include "sampling.cuh"

namespace {

using namespace qmk_sample;

int refuse(const std::string &why) {
  qmk_internal::note_error("qmk_sample_tokens: " + why);
  return QMK_ERR_BAD_ARGUMENT;
}

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
cudaError_t launch(const Params &p, int rows, cudaStream_t stream) {
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

}  // namespace

extern "C" int qmk_sample_tokens(const void *logits, int logits_type, long long row_stride, int rows, int vocab, const float *uniforms,
                                 const float *temperatures, float temperature, const int *top_ks, int top_k, const float *top_ps,
                                 float top_p, const float *min_ps, float min_p, int *tokens, float *logprobs, cudaStream_t stream) {
  qmk_internal::begin_call();
  if (rows == 0) return QMK_OK;
  if (rows < 0 || rows > 1 << 16) return refuse("rows must be in [0, 65536]");
  if (vocab < 1 || vocab > MAX_VOCAB) return refuse("the vocabulary must be in [1, 262144]");
  if (logits_type < 0 || logits_type > 2) return refuse("logits are fp32 (0), fp16 (1) or bf16 (2)");
  if (!logits || !uniforms || !tokens) return refuse("null pointer argument");
  if (rows > 1 && row_stride < vocab && row_stride != 0) return refuse("rows overlap: the row stride is below the vocabulary");
  if (!temperatures && !(temperature >= 0.0f)) return refuse("the temperature must not be negative");
  if (!top_ps && !(top_p > 0.0f)) return refuse("top_p must be above 0");
  if (!min_ps && !(min_p >= 0.0f && min_p <= 1.0f)) return refuse("min_p must be in [0, 1]");
  Params p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.uniforms = uniforms;
  p.temperatures = temperatures;
  p.top_ps = top_ps;
  p.min_ps = min_ps;
  p.top_ks = top_ks;
  p.temperature = temperature;
  p.top_p = top_p;
  p.min_p = min_p;
  p.top_k = top_k;
  p.tokens = tokens;
  p.logprobs = logprobs;
  const cudaError_t e = logits_type == 0 ? launch<float>(p, rows, stream) : logits_type == 1 ? launch<__half>(p, rows, stream) : launch<__nv_bfloat16>(p, rows, stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    qmk_internal::note_error(std::string("qmk_sample_tokens: ") + cudaGetErrorString(e));
    return QMK_ERR_CUDA;
  }
  return QMK_OK;
}
