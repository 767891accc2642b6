// C entry of the sampling kernel (sampling.cuh).
#include "../../include/qwen_megakernel.h"

#include <string>

#include "engine_internal.h"
#include "sampling.cuh"

namespace {

using namespace qmk_sample;

int refuse(const std::string &why) {
  qmk_internal::note_error("qmk_sample_tokens: " + why);
  return QMK_ERR_BAD_ARGUMENT;
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
  if (reinterpret_cast<unsigned long long>(logits) % (logits_type == 0 ? 4 : 2)) return refuse("the logits' address must be aligned to their size");
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
  const cudaError_t e = logits_type == 0 ? launch_fp32(p, rows, stream) : logits_type == 1 ? launch_fp16(p, rows, stream) : launch_bf16(p, rows, stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    qmk_internal::note_error(std::string("qmk_sample_tokens: ") + cudaGetErrorString(e));
    return QMK_ERR_CUDA;
  }
  return QMK_OK;
}
