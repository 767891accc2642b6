// C entry of the sampling kernel (sampling.cuh).
#include "../../include/qwen_megakernel.h"

#include <algorithm>
#include <string>

#include "engine_internal.h"
#include "sampling.cuh"

namespace {

using namespace qmk_sample;

int refuse(const std::string &why) {
  qmk_internal::note_error("qmk_sample_tokens: " + why);
  return QMK_ERR_BAD_ARGUMENT;
}

// CTAs per row: as many as still are all resident at once (two an SM), each with 2048 tokens at least.
int cluster_size(int rows, int vocab, int sms) {
  int c = 1;
  while (c < MAX_CLUSTER && 2 * c * rows <= 2 * sms && vocab > c * 2048) c *= 2;
  return c;
}

template <typename T>
cudaError_t launch(const Params &p, int rows, int ranks, int sms, cudaStream_t stream) {
  void (*const kernel)(Params) = rows * ranks <= sms ? sample_rows<T, 1> : sample_rows<T, 2>;
  constexpr int smem = sizeof(Shared) + 2 * TURN * THREADS * 4 * sizeof(T);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = dim3(static_cast<unsigned int>(rows) * ranks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
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
  if (rows > 1 && row_stride < vocab) return refuse("rows overlap: the row stride is below the vocabulary");
  if (!temperatures && !(temperature >= 0.0f)) return refuse("the temperature must not be negative");
  if (!top_ps && !(top_p > 0.0f)) return refuse("top_p must be above 0");
  if (!min_ps && !(min_p >= 0.0f && min_p <= 1.0f)) return refuse("min_p must be in [0, 1]");
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) {
    cudaGetLastError();
    qmk_internal::note_error(std::string("qmk_sample_tokens: ") + cudaGetErrorString(e));
    return QMK_ERR_CUDA;
  }
  Params p;
  const int ranks = cluster_size(rows, vocab, sms);
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
  e = logits_type == 0 ? launch<float>(p, rows, ranks, sms, stream)
      : logits_type == 1 ? launch<__half>(p, rows, ranks, sms, stream)
                         : launch<__nv_bfloat16>(p, rows, ranks, sms, stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    qmk_internal::note_error(std::string("qmk_sample_tokens: ") + cudaGetErrorString(e));
    return QMK_ERR_CUDA;
  }
  return QMK_OK;
}
