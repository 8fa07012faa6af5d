// Token sampling from logits (include/qwen_b200_ops.h has the definition).
#pragma once

#include <cuda_runtime.h>

namespace qb {
namespace sampling {

constexpr int kMaxVocab = 1 << 18;

// Row r of the logits starts at logits + r * stride elements. Each setting may be null (off; temperature: 1).
struct Sample {
  const void* logits;
  int rows, vocab;
  long long stride;
  const float* temperature;
  const int* top_k;
  const float *top_p, *min_p, *uniforms;
  int* tokens;
  float* probs;  // may be null
};

cudaError_t launch_sample(const Sample& a, int type, cudaStream_t s);

}  // namespace sampling
}  // namespace qb
