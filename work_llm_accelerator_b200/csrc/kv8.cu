// Writing rows into the 8-bit KV cache and reading them back (include/qwen_b200_ops.h).
//
// One CTA takes one block of 64 tokens of one sequence and kv head: a block has one scale, so the CTA that owns
// it sees every value that the scale depends on and no two CTAs write the same bytes. Both kernels are bound by
// the bytes they move, small calls by the chain of loads that finds a CTA's block (segments, block table, data); each
// value is loaded once, kept in registers while the CTA agrees on the scale, and stored once.
// Measured on B200, 2 kv heads: append of 64 single rows 3.3 us, of 4096 fp32 rows 4.1 us, of 18400 bf16 rows in ragged
// chunks 10.1 us (28 MB); read of 32768 fp32 rows 16.9 us (84 MB, 5.0 TB/s).
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
  int block, first_slot, n;  // block: id in the cache, -1: no such block; slots first_slot .. first_slot + n - 1
  long long row;             // row of first_slot
};

// Unit u -> (segment, block). Segment i with c rows touches at most floor(c / 64) + 2 blocks, so it gets the units
// from floor(offsets[i] / 64) + 2 i on: those starts leave it room for that many, and there are
// n_rows / 64 + 2 * segments in all. The segment is found by counting the starts that are not above u; the thread that
// holds its numbers finds the block and tells the others.
__device__ __forceinline__ bool find_work(const Cache& c, const Rows& r, int u, Work& out) {
  __shared__ Work w;
  for (int base = 0; base < r.segments; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    const bool in = i < r.segments;
    const int lo = in ? __ldg(r.offsets + i) : 0, hi = in ? __ldg(r.offsets + i + 1) : 0;
    const int start = in ? __ldg(r.starts + i) : 0, seq = in ? __ldg(r.seqs + i) : 0;
    const int first = lo / kBlock + 2 * i;
    const int n = __syncthreads_count(in && first <= u);
    if (n == kThreads && base + kThreads < r.segments && __ldg(r.offsets + base + kThreads) / kBlock + 2 * (base + kThreads) <= u)
      continue;
    if (n == 0) return false;  // only where offsets do not begin at 0
    if ((int)threadIdx.x == n - 1) {
      w.n = 0;
      const int j = u - first;
      const long long end = (long long)start + (hi - lo);
      if (lo != hi) {
        if (lo < 0 || hi < lo || hi > r.n_rows || start < 0 || seq < 0 || seq >= c.n_seqs || j < 0 ||
            end > (long long)c.width * kBlock) {
          bad_index();
        } else if (start / kBlock + (long long)j < c.width) {
          const int blk = start / kBlock + j;
          const int from = max(start, blk * kBlock), to = (int)min(end, ((long long)blk + 1) * kBlock);
          if (from < to) {
            w.first_slot = from % kBlock;
            w.n = to - from;
            w.row = lo + (from - start);
            const int block = __ldg(c.table + (long long)seq * c.width + blk);
            w.block = block;
            if (block < 0 || block >= c.n_blocks) {
              bad_index();
              w.block = -1;
            }
          }
        }
      }
    }
    __syncthreads();
    out = w;
    return out.n > 0;
  }
  return false;
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

// Four codes rint(fl(x / s)), r = fl(1 / s). x r is off by at most 2^-23 of it, the quotient by 2^-24, and neither is above
// 127 (1 + 2^-22), so both round to the same integer unless x r lies within 127 * 2^-22.4 = 2.3e-5 of the middle between
// two: those few take the division. Adding 1.5 * 2^23 rounds to even and leaves the code in the low byte.
__device__ __forceinline__ unsigned codes_of(float4 x, float s, float r) {
  constexpr float kRound = 12582912.0f, kMiddle = 0.5f - 4e-5f;
  const float4 t = make_float4(x.x * r, x.y * r, x.z * r, x.w * r);
  const float4 n = make_float4(t.x + kRound, t.y + kRound, t.z + kRound, t.w + kRound);
  const float d = fmaxf(fmaxf(fabsf(t.x - (n.x - kRound)), fabsf(t.y - (n.y - kRound))),
                        fmaxf(fabsf(t.z - (n.z - kRound)), fabsf(t.w - (n.w - kRound))));
  if (d > kMiddle)
    return (code_of(x.x, s) & 0xff) | (code_of(x.y, s) & 0xff) << 8 | (code_of(x.z, s) & 0xff) << 16 | (unsigned)code_of(x.w, s) << 24;
  return __byte_perm(__byte_perm(__float_as_uint(n.x), __float_as_uint(n.y), 0x0040),
                     __byte_perm(__float_as_uint(n.z), __float_as_uint(n.w), 0x0040), 0x5410);
}

__device__ __forceinline__ unsigned abs_bits(float4 v) {
  return max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
             max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
}

// K and V in CTAs of their own, 16-bit values packed until they are used: with both in one CTA, its registers leave room
// for two per SM and 18400 bf16 rows took 16.2 us; apart 11.7, packed 10.1.
template <int kType>
__global__ void __launch_bounds__(kThreads, kType == 0 ? 4 : kType == 1 ? 5 : 6) append_kernel(Cache c, const void* k, const void* v, Rows r) {
  using T = typename TypeOf<kType>::T;
  __shared__ unsigned warp_max[kWarps];
  Work w;
  if (!find_work(c, r, blockIdx.x, w) || w.block < 0) return;
  const int head = blockIdx.y, which = blockIdx.z, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long at = (long long)w.block * c.heads + head;
  const T* x = static_cast<const T*>(which ? v : k) + w.row * r.stride + head * kHead + lane * 4;
  float* scale = (which ? c.scales[1] : c.scales[0]) + at;
  int* codes = reinterpret_cast<int*>((which ? c.codes[1] : c.codes[0]) + at * kBlock * kHead) + lane;
  const bool opened = w.first_slot > 0;
  const float old = opened ? *scale : 0.0f;

  decltype(raw4(x)) val[kSlotsPerWarp];
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    val[i] = {};
    if (t < w.n) val[i] = raw4(x + t * r.stride);
  }
  unsigned a = 0;  // absolute values compare as their bits; NaN and infinities are the largest
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) a = max(a, abs_bits(expand<T>(val[i])));
  a = __reduce_max_sync(0xffffffffu, a);
  if (lane == 0) warp_max[warp] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) a = max(a, warp_max[i]);
  int twice;
  const float s = grown_scale(a, opened, old, twice);
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
  const float inv = 1.0f / s;
  codes += (w.first_slot + warp) * (kHead / 4);
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i)
    if (warp + i * kWarps < w.n) codes[i * kWarps * (kHead / 4)] = zero ? 0 : codes_of(expand<T>(val[i]), s, inv);
}

__device__ __forceinline__ float4 values_of(int b, float s) {
  return make_float4((float)(int8_t)b * s, (float)(int8_t)(b >> 8) * s, (float)(int8_t)(b >> 16) * s, (float)(b >> 24) * s);
}

template <int kType>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache c, void* k, void* v, Rows r) {
  using T = typename TypeOf<kType>::T;
  Work w;
  if (!find_work(c, r, blockIdx.x, w)) return;
  const int head = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long to = w.row * r.stride + head * kHead + lane * 4;
  T* x = static_cast<T*>(k) + to;
  T* y = static_cast<T*>(v) + to;
  const bool bad = w.block < 0;
  const long long at = (long long)max(w.block, 0) * c.heads + head, from = at * kBlock * kHead + w.first_slot * kHead + lane * 4;
  const int* kc = reinterpret_cast<const int*>(c.codes[0] + from);
  const int* vc = reinterpret_cast<const int*>(c.codes[1] + from);
  int kb[kSlotsPerWarp], vb[kSlotsPerWarp];
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    kb[i] = t < w.n ? kc[t * (kHead / 4)] : 0;
    vb[i] = t < w.n ? vc[t * (kHead / 4)] : 0;
  }
  // a block id outside of the cache reads as NaN
  const float nan = __int_as_float(0x7fc00000), ks = bad ? nan : c.scales[0][at], vs = bad ? nan : c.scales[1][at];
#pragma unroll
  for (int i = 0; i < kSlotsPerWarp; ++i) {
    const int t = warp + i * kWarps;
    if (t >= w.n) break;
    stream4(x + t * r.stride, values_of(kb[i], ks));
    stream4(y + t * r.stride, values_of(vb[i], vs));
  }
}

dim3 grid_of(const Cache& c, const Rows& r, unsigned z) {
  return dim3((unsigned)(r.n_rows / kBlock + 2 * (long long)r.segments), (unsigned)c.heads, z);
}

}  // namespace

cudaError_t launch_append(const Cache& c, const void* k, const void* v, int type, const Rows& r, cudaStream_t s) {
  const dim3 grid = grid_of(c, r, 2);
  if (type == 0) append_kernel<0><<<grid, kThreads, 0, s>>>(c, k, v, r);
  else if (type == 1) append_kernel<1><<<grid, kThreads, 0, s>>>(c, k, v, r);
  else append_kernel<2><<<grid, kThreads, 0, s>>>(c, k, v, r);
  return cudaGetLastError();
}

cudaError_t launch_read(const Cache& c, void* k, void* v, int type, const Rows& r, cudaStream_t s) {
  const dim3 grid = grid_of(c, r, 1);
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
