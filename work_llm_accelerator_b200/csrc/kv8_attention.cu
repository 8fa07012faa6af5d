// Decode attention over the 8-bit KV cache (include/qwen_b200_ops.h): one query row per new token, the row's
// own length, softmax in one pass with the running maximum and sum in fp32.
//
// The cache's scales leave the sums: with k_j = s_k c_j a score is (scale s_k) (q . c_j).
// A tile of 64 tokens is summed by itself, relative to its own maximum, and then joined to the running sums:
// weights far below the row's largest one are not rounded away one by one against a large sum.
// Simple form: one CTA per query row and head, a warp per tile, four dimensions per lane.
#include <cuda_runtime.h>

#include "kv8_device.cuh"

namespace qb {
namespace kv8 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

template <int kType>
__global__ void __launch_bounds__(kThreads) attention_kernel(Cache c, Attend a) {
  using T = typename TypeOf<kType>::T;
  __shared__ float part[kWarps][kHead], top[kWarps], sum[kWarps];
  const int row = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int seq = a.row_seq[row];
  if (seq < 0) return;
  const int len = a.row_len[row];
  const float nan = __int_as_float(0x7fc00000);
  const bool bad = seq >= c.n_seqs || len < 0 || len > (long long)c.width * kBlock;
  if (bad && threadIdx.x == 0) bad_index();
  const int head = h / (a.q_heads / c.heads);
  const float4 q = load4(static_cast<const T*>(a.q) + row * a.q_stride + h * kHead + lane * 4);
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int tile = warp * kBlock; !bad && tile < len; tile += kWarps * kBlock) {
    const int block = c.table[(long long)seq * c.width + tile / kBlock];
    const bool out = block < 0 || block >= c.n_blocks;
    if (out) bad_index();
    const long long at = (long long)(out ? 0 : block) * c.heads + head;
    const float ks = out ? nan : c.scales[0][at], vs = out ? nan : c.scales[1][at];
    float tm = -INFINITY, tl = 0.0f;
    float4 to = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = 0; t < min(kBlock, len - tile); ++t) {
      const long long off = (at * kBlock + t) * kHead + lane * 4;
      const char4 k = *reinterpret_cast<const char4*>(c.codes[0] + off);
      const char4 v = *reinterpret_cast<const char4*>(c.codes[1] + off);
      float d = fmaf(q.x, (float)k.x, fmaf(q.y, (float)k.y, fmaf(q.z, (float)k.z, q.w * (float)k.w)));
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) d += __shfl_xor_sync(0xffffffffu, d, i);
      const float s = d * (a.scale * ks);
      const float n = s > tm ? s : (s == s ? tm : s);  // a NaN stays
      const float keep = tm == n ? 1.0f : expf(tm - n), p = expf(s - n);
      tm = n;
      tl = tl * keep + p;
      to = make_float4(fmaf(p, (float)v.x, to.x * keep), fmaf(p, (float)v.y, to.y * keep),
                       fmaf(p, (float)v.z, to.z * keep), fmaf(p, (float)v.w, to.w * keep));
    }
    const float n = tm > m ? tm : (tm == tm ? m : tm);
    const float keep = m == n ? 1.0f : expf(m - n), add = tm == n ? 1.0f : expf(tm - n), av = add * vs;
    m = n;
    l = l * keep + add * tl;
    o = make_float4(fmaf(av, to.x, o.x * keep), fmaf(av, to.y, o.y * keep), fmaf(av, to.z, o.z * keep),
                    fmaf(av, to.w, o.w * keep));
  }
  if (lane == 0) {
    top[warp] = m;
    sum[warp] = l;
  }
  *reinterpret_cast<float4*>(&part[warp][lane * 4]) = o;
  __syncthreads();
  if (warp != 0) return;
  float best = -INFINITY, total = 0.0f;
  for (int w = 0; w < kWarps; ++w) best = top[w] > best ? top[w] : (top[w] == top[w] ? best : top[w]);
  o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int w = 0; w < kWarps; ++w) {
    if (sum[w] == 0.0f) continue;
    const float f = expf(top[w] - best);
    const float4 p = *reinterpret_cast<float4*>(&part[w][lane * 4]);
    total += f * sum[w];
    o = make_float4(fmaf(f, p.x, o.x), fmaf(f, p.y, o.y), fmaf(f, p.z, o.z), fmaf(f, p.w, o.w));
  }
  const float r = bad ? nan : total == 0.0f ? 0.0f : 1.0f / total;
  store4(static_cast<T*>(a.out) + row * a.out_stride + h * kHead + lane * 4, make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
  if (a.lse && lane == 0) a.lse[(long long)row * a.q_heads + h] = bad ? nan : best + logf(total);
}

}  // namespace

size_t attention_workspace(int, int, int) { return 256; }

cudaError_t launch_attention(const Cache& c, const Attend& a, int type, cudaStream_t s) {
  const dim3 grid((unsigned)a.rows, (unsigned)a.q_heads);
  if (type == 0) attention_kernel<0><<<grid, kThreads, 0, s>>>(c, a);
  else if (type == 1) attention_kernel<1><<<grid, kThreads, 0, s>>>(c, a);
  else attention_kernel<2><<<grid, kThreads, 0, s>>>(c, a);
  return cudaGetLastError();
}

unsigned attention_kernel_error(bool reset) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_kernel_error, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
  if (reset) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(g_kernel_error, &z, sizeof(z));
  }
  return v;
}

}  // namespace kv8
}  // namespace qb
