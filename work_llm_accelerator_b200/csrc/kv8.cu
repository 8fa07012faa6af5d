// Writing rows into the 8-bit KV cache and reading them back (include/qwen_b200_ops.h).
//
// One CTA takes one block of 64 tokens of one sequence and kv head (and K or V, when it writes): a block has one
// scale, so the CTA that owns it sees every value that the scale depends on and no two CTAs write the same
// bytes. Both kernels are bound by the bytes they move; each value is loaded once, kept in registers while
// the CTA agrees on the scale, and stored once.
#include <cuda_runtime.h>

#include "kv8_device.cuh"

namespace qb {
namespace kv8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSlotsPerWarp = kBlock / kWarps;

// The rows of one block that a CTA works on.
struct Work {
  int seq, block, first_slot, n;  // block: id in the cache; slots first_slot .. first_slot + n - 1
  long long row;                  // row of first_slot
  bool opened;                    // the block holds earlier tokens of the sequence
};

// Unit u -> (segment, block). Segment i with c rows touches at most floor(c / 64) + 2 blocks, so it gets the units
// from floor(offsets[i] / 64) + 2 i on: those starts leave it room for that many, and there are
// n_rows / 64 + 2 * segments in all. The segment is found by counting the starts that are not above u.
__device__ __forceinline__ bool find_work(const Cache& c, const Rows& r, int u, Work& w) {
  int seg = -1;
  for (int base = 0; base < r.segments; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    const bool before = i < r.segments && r.offsets[i] / kBlock + 2 * i <= u;
    const int n = __syncthreads_count(before);
    seg += n;
    if (n < kThreads) break;
  }
  if (seg < 0) return false;
  const int lo = r.offsets[seg], hi = r.offsets[seg + 1], start = r.starts[seg], seq = r.seqs[seg];
  const int j = u - (lo / kBlock + 2 * seg);
  if (lo == hi) return false;
  if (lo < 0 || hi < lo || hi > r.n_rows || start < 0 || seq < 0 || seq >= c.n_seqs || j < 0 ||
      (long long)start + (hi - lo) > (long long)c.width * kBlock) {
    if (threadIdx.x == 0) bad_index();
    return false;
  }
  const int blk = start / kBlock + j;
  const int from = max(start, blk * kBlock), to = (int)min((long long)start + (hi - lo), ((long long)blk + 1) * kBlock);
  if (from >= to) return false;
  w.seq = seq;
  w.first_slot = from % kBlock;
  w.n = to - from;
  w.row = lo + (from - start);
  w.opened = w.first_slot > 0;
  w.block = c.table[(long long)seq * c.width + blk];
  if (w.block < 0 || w.block >= c.n_blocks) {
    if (threadIdx.x == 0) bad_index();
    w.block = -1;
  }
  return true;
}

// The scale of a block after values of at most `a` (the bits of an fp32 absolute value) come to it.
//   opened by this call: need = a * fl(1 / 127), at least 2^-126 (a subnormal scale would not give 127 steps)
//   held tokens already: the old scale, doubled until it is at least need. Halving the older codes as often rounds
//   them to half a step of the new scale, so with the final scale s all roundings of a value together stay below
//   s/2 (1 + 1/2 + 1/4 + ...) = s. Growing to need itself could round the older codes up to 63 times, by s/2 each.
__device__ __forceinline__ float grown_scale(unsigned a, bool opened, float old, int& twice) {
  twice = 0;
  const float nan = __int_as_float(0x7fc00000);
  if (a >= 0x7f800000u) return nan;  // a NaN or an infinity: the whole block reads as NaN
  const float need = a == 0 ? 0.0f : fmaxf(__uint_as_float(a) * (1.0f / 127.0f), 1.17549435e-38f);
  if (!opened || old == 0.0f) return need;  // a scale of zero: every older code is zero
  if (!(old > 0.0f) || old > 3.4e38f) return nan;
  if (need <= old) return old;
  int e1, e2;
  const float m1 = frexpf(need, &e1), m2 = frexpf(old, &e2);
  twice = e1 - e2 + (m1 > m2 ? 1 : 0);
  return ldexpf(old, twice);
}

__device__ __forceinline__ int code_of(float x, float s) {
  return max(-127, min(127, __float2int_rn(__fdiv_rn(x, s))));
}

template <int kType>
__global__ void __launch_bounds__(kThreads) append_kernel(Cache c, const void* k, const void* v, Rows r) {
  using T = typename TypeOf<kType>::T;
  __shared__ unsigned warp_max[kWarps];
  Work w;
  if (!find_work(c, r, blockIdx.x, w) || w.block < 0) return;
  const int head = blockIdx.y, which = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const T* x = static_cast<const T*>(which ? v : k) + w.row * r.stride + head * kHead + lane * 4;
  const long long at = (long long)w.block * c.heads + head;
  float* scale = c.scales[which] + at;
  int* codes = reinterpret_cast<int*>(c.codes[which] + at * kBlock * kHead) + lane;
  const float old = w.opened ? *scale : 0.0f;

  float4 val[kSlotsPerWarp];
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    val[i] = t < w.n ? load4(x + t * r.stride) : make_float4(0.f, 0.f, 0.f, 0.f);
    // absolute values compare as their bits; NaN and infinities are the largest
    a = max(a, max(max(__float_as_uint(val[i].x) & 0x7fffffffu, __float_as_uint(val[i].y) & 0x7fffffffu),
                   max(__float_as_uint(val[i].z) & 0x7fffffffu, __float_as_uint(val[i].w) & 0x7fffffffu)));
  }
  a = __reduce_max_sync(0xffffffffu, a);
  if (lane == 0) warp_max[warp] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) a = max(a, warp_max[i]);
  int twice;
  const float s = grown_scale(a, w.opened, old, twice);
  if (threadIdx.x == 0) *scale = s;
  if (twice > 0) {
    const float half = ldexpf(1.0f, -twice);
    for (int t = warp; t < w.first_slot; t += kWarps) {
      const int b = codes[t * (kHead / 4)];
      int n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) n |= (__float2int_rn((float)(int8_t)(b >> (8 * i)) * half) & 0xff) << (8 * i);
      codes[t * (kHead / 4)] = n;
    }
  }
  const bool zero = !(s > 0.0f);  // all zero, or NaN
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    if (t >= w.n) break;
    int n = 0;
    if (!zero)
      n = (code_of(val[i].x, s) & 0xff) | (code_of(val[i].y, s) & 0xff) << 8 | (code_of(val[i].z, s) & 0xff) << 16 |
          code_of(val[i].w, s) << 24;
    codes[(w.first_slot + t) * (kHead / 4)] = n;
  }
}

template <int kType>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache c, void* k, void* v, Rows r) {
  using T = typename TypeOf<kType>::T;
  Work w;
  if (!find_work(c, r, blockIdx.x, w)) return;
  const int head = blockIdx.y, which = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  T* x = static_cast<T*>(which ? v : k) + w.row * r.stride + head * kHead + lane * 4;
  const long long at = (long long)max(w.block, 0) * c.heads + head;
  // a block id outside of the cache reads as NaN
  const float s = w.block < 0 ? __int_as_float(0x7fc00000) : c.scales[which][at];
  const int* codes = reinterpret_cast<const int*>(c.codes[which] + at * kBlock * kHead) + w.first_slot * (kHead / 4) + lane;
  int b[kSlotsPerWarp];
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    b[i] = t < w.n && w.block >= 0 ? codes[t * (kHead / 4)] : 0;
  }
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    if (t < w.n)
      store4(x + t * r.stride, make_float4((float)(int8_t)b[i] * s, (float)(int8_t)(b[i] >> 8) * s,
                                           (float)(int8_t)(b[i] >> 16) * s, (float)(b[i] >> 24) * s));
  }
}

dim3 grid_of(const Cache& c, const Rows& r) {
  return dim3((unsigned)(r.n_rows / kBlock + 2 * (long long)r.segments), (unsigned)c.heads, 2);
}

}  // namespace

cudaError_t launch_append(const Cache& c, const void* k, const void* v, int type, const Rows& r, cudaStream_t s) {
  const dim3 grid = grid_of(c, r);
  if (type == 0) append_kernel<0><<<grid, kThreads, 0, s>>>(c, k, v, r);
  else if (type == 1) append_kernel<1><<<grid, kThreads, 0, s>>>(c, k, v, r);
  else append_kernel<2><<<grid, kThreads, 0, s>>>(c, k, v, r);
  return cudaGetLastError();
}

cudaError_t launch_read(const Cache& c, void* k, void* v, int type, const Rows& r, cudaStream_t s) {
  const dim3 grid = grid_of(c, r);
  if (type == 0) read_kernel<0><<<grid, kThreads, 0, s>>>(c, k, v, r);
  else if (type == 1) read_kernel<1><<<grid, kThreads, 0, s>>>(c, k, v, r);
  else read_kernel<2><<<grid, kThreads, 0, s>>>(c, k, v, r);
  return cudaGetLastError();
}

unsigned kernel_error(bool reset) {
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
