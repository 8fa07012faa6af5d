// Sampling with temperature, top-k, top-p and min-p from given uniform numbers (include/qwen_b200_ops.h).
//
// A row's tokens are ordered by logit, ties by index. Both go into one integer, `order` = the logit's bits made
// monotone, then the complement of the index, so the order is strict and every set that the filters keep is
// { order >= some threshold }. Simple form: one CTA per row, each threshold by bisection over the bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "sample.h"

namespace qb {
namespace sampling {
namespace {

constexpr int kThreads = 1024;

template <int kType>
__device__ __forceinline__ float load(const void* p, long long i);
template <>
__device__ __forceinline__ float load<0>(const void* p, long long i) {
  return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float load<1>(const void* p, long long i) {
  return __half2float(static_cast<const __half*>(p)[i]);
}
template <>
__device__ __forceinline__ float load<2>(const void* p, long long i) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ unsigned long long order_of(float x, int i) {
  const unsigned b = __float_as_uint(x + 0.0f);  // -0 becomes +0: they tie
  const unsigned up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)up << 18 | (unsigned)(kMaxVocab - 1 - i);
}

// Sums over the CTA in a fixed order.
struct Totals {
  long long n;
  double w;
};
__device__ Totals cta_sum(Totals t) {
  __shared__ Totals part[kThreads / 32];
  for (int i = 16; i > 0; i >>= 1) {
    t.n += __shfl_xor_sync(0xffffffffu, t.n, i);
    t.w += __shfl_xor_sync(0xffffffffu, t.w, i);
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = t;
  __syncthreads();
  t = {0, 0.0};
  for (int i = 0; i < kThreads / 32; ++i) {
    t.n += part[i].n;
    t.w += part[i].w;
  }
  return t;
}

template <int kType>
__global__ void __launch_bounds__(kThreads) sample_kernel(Sample a) {
  const int row = blockIdx.x;
  const long long base = (long long)row * a.stride;
  __shared__ unsigned long long best_s;
  if (threadIdx.x == 0) best_s = 0;
  __syncthreads();
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float x = load<kType>(a.logits, base + i);
    if (x > -INFINITY) best = max(best, order_of(x, i));
  }
  atomicMax(&best_s, best);
  __syncthreads();
  best = best_s;
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const int first = kMaxVocab - 1 - (int)(best & (kMaxVocab - 1));
  if (best == 0 || !(temp >= 1.17549435e-38f)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = best == 0 ? -1 : first;
      if (a.probs) a.probs[row] = best == 0 ? 0.0f : 1.0f;
    }
    return;
  }
  const double top = load<kType>(a.logits, base + first);
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
  auto weight = [&](float x) { return x == top ? 1.0 : exp(((double)x - top) / (double)temp); };
  unsigned long long keep = 1;  // the kept set: order >= keep, and weight >= least
  double least = 0.0;
  auto sums = [&](unsigned long long from) {
    Totals t{0, 0.0};
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const float x = load<kType>(a.logits, base + i);
      if (!(x > -INFINITY)) continue;
      const unsigned long long o = order_of(x, i);
      if (o < from || o < keep) continue;
      const double w = weight(x);
      if (w < least && o != best) continue;
      t.n++;
      t.w += w;
    }
    return cta_sum(t);
  };
  // the largest threshold whose set satisfies `enough`, 0 if none does
  auto largest = [&](auto enough) {
    unsigned long long c = 0;
    for (int bit = 49; bit >= 0; --bit)
      if (enough(sums(c | 1ull << bit))) c |= 1ull << bit;
    return c;
  };
  if (k > 0 && k < a.vocab) keep = max(keep, largest([&](Totals t) { return t.n >= k; }));
  if (p < 1.0f) {
    const double want = (double)p * sums(0).w;
    const unsigned long long c = largest([&](Totals t) { return t.w >= want && t.n > 0; });
    keep = max(keep, c);
  }
  least = mp;
  const double total = sums(0).w;
  const float u = a.uniforms[row];
  const double want = (u > 0.0f ? (double)u : 0.0) * total;
  unsigned long long c = largest([&](Totals t) { return t.w > want; });
  if (c == 0) {  // u = 1: the last one kept
    const long long n = sums(0).n;
    c = largest([&](Totals t) { return t.n >= n; });
  }
  if (threadIdx.x == 0) {
    const int token = kMaxVocab - 1 - (int)(c & (kMaxVocab - 1));
    a.tokens[row] = token;
    if (a.probs) a.probs[row] = (float)(weight(load<kType>(a.logits, base + token)) / total);
  }
}

}  // namespace

cudaError_t launch_sample(const Sample& a, int type, cudaStream_t s) {
  if (type == 0) sample_kernel<0><<<a.rows, kThreads, 0, s>>>(a);
  else if (type == 1) sample_kernel<1><<<a.rows, kThreads, 0, s>>>(a);
  else sample_kernel<2><<<a.rows, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace sampling
}  // namespace qb
