// Sampling with temperature, top-k, top-p and min-p from given uniform numbers (include/qwen_b200_ops.h).
//
// A row's tokens are ordered by logit, ties by index. Both go into one integer, `order` = the logit's bits made
// monotone, then the complement of the index, so the order is strict and what each filter keeps is a prefix of it.
//
// No row is sorted. With z = (max - logit) / temperature a token weighs w = exp(-z). Its bucket is b = floor(64 z)
// (2048 of them; beyond z = 32 a weight is below 1.3e-14 of the first token's and counts as 0), and inside its bucket
// w = exp(-b/64) (1 - q 2^-23) with the integer q = rint(2^23 (1 - exp(-f))), f = z - b/64. One pass adds up the
// count and the q of every bucket, as integers, so neither the sums nor the token depend on the order of the
// atomics. The bucket sums (in 64 bits) tell in which bucket each filter's border and the drawn number fall, and only
// tokens of such buckets are gathered and sorted. A weight is off by the
// rounding of q, 2^-24 of its bucket's largest, and by that of max - logit, z 2^-24 of itself, both at random: 1 /
// temperature is held to 2^-48, so that no error is common to all weights, which a number drawn among 150000 small ones
// needs.
//
// A row is read three times: for its maximum, for the bucket sums, for the tokens to sort; the second and third reading
// mostly meet L2. A cluster of 8 CTAs shares a row while each finds an SM of its own, one of 4, 2 or 1 while all run at
// once, two per SM. The first CTA leads: it gets the others' bucket sums through distributed shared memory, decides (every
// warp the same way, without barriers) and asks for what it needs to see. Bound: for few rows
// the latency of those steps, for many the two shared atomics per logit of the second pass (4.1 cycles each at random
// banks). Measured on B200, vocabulary 151936: 1 fp32 row with all filters 19.0 us, 64 rows with settings of their own
// 65.3 us, 256 bf16 rows without filters 120 us. Two CTAs per SM leave 64 registers, of which the leader's part spills
// 0.6 to 1 KB; with 128 and one CTA per SM 64 rows take 78 us and 256 rows 124 (but 150 rows 114 instead of 139).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "qwen_common.cuh"
#include "sample.h"

namespace cg = cooperative_groups;

namespace qb {
namespace sampling {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBuckets = 2048;
constexpr int kPerThread = kBuckets / kThreads;
constexpr int kList = 2048;  // tokens that are sorted at once
constexpr int kOrderBits = 50;
constexpr int kDigit = 11;        // bits by which a crowded bucket is narrowed at a time
constexpr int kFold = 1 << 15;    // logits whose q, below 2^17 each, fit a 32-bit sum
constexpr int kAhead = 4;         // 16-byte loads that a thread has under way (8 cost registers: 256 rows took 9% longer)
constexpr int kMaxCluster = 8;
constexpr int kOneCta = 8192;     // vocabularies up to this size take one CTA: less to read than a cluster costs to sync
constexpr int kSms = 148;

typedef unsigned long long u64;

// A type's values: one from memory, and the kVec ones of 16 bytes (by bit operations, so that they stay in registers).
template <int kType>
struct TypeOf;
template <>
struct TypeOf<0> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float one(const T* p) { return __ldg(p); }
  static __device__ __forceinline__ void unpack(const uint4& b, float (&v)[kVec]) {
    v[0] = __uint_as_float(b.x), v[1] = __uint_as_float(b.y), v[2] = __uint_as_float(b.z), v[3] = __uint_as_float(b.w);
  }
};
template <>
struct TypeOf<1> {
  using T = __half;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(const T* p) { return __half2float(*p); }
  static __device__ __forceinline__ float half_at(unsigned w, int hi) {
    return __half2float(__ushort_as_half((unsigned short)(hi ? w >> 16 : w & 0xffffu)));
  }
  static __device__ __forceinline__ void unpack(const uint4& b, float (&v)[kVec]) {
    v[0] = half_at(b.x, 0), v[1] = half_at(b.x, 1), v[2] = half_at(b.y, 0), v[3] = half_at(b.y, 1);
    v[4] = half_at(b.z, 0), v[5] = half_at(b.z, 1), v[6] = half_at(b.w, 0), v[7] = half_at(b.w, 1);
  }
};
template <>
struct TypeOf<2> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(const T* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& b, float (&v)[kVec]) {
    v[0] = __uint_as_float(b.x << 16), v[1] = __uint_as_float(b.x & 0xffff0000u);
    v[2] = __uint_as_float(b.y << 16), v[3] = __uint_as_float(b.y & 0xffff0000u);
    v[4] = __uint_as_float(b.z << 16), v[5] = __uint_as_float(b.z & 0xffff0000u);
    v[6] = __uint_as_float(b.w << 16), v[7] = __uint_as_float(b.w & 0xffff0000u);
  }
};

__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 order_of(float x, int i) { return (u64)key_of(x) << 18 | (unsigned)(kMaxVocab - 1 - i); }
__device__ __forceinline__ int index_of(u64 order) { return kMaxVocab - 1 - (int)(order & (kMaxVocab - 1)); }
__device__ __forceinline__ float value_of(u64 order) { return value_of((unsigned)(order >> 18)); }

__device__ __forceinline__ F2 add2_down(F2 a, F2 b) {
  F2 r;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// 64 z = 64 (top - x) / temperature in parts: bucket and q. 64 / temperature = c + c_low to 2^-48, so that no error is
// common to all weights; the difference top - x is rounded to fp32.
struct Scale {
  float top, c, c_low;
  __device__ Scale() {}
  __device__ Scale(float top_, float t) : top(top_) {
    const float r = 1.0f / t;
    float low = r > 0.0f ? fmaf(-t, r, 1.0f) * r : 0.0f;
    if (!(fabsf(low) < r)) low = 0.0f;
    c = 64.0f * r;
    c_low = 64.0f * low;
  }
  static constexpr float kFloor = 8388608.0f;  // 2^23: added rounding down, the sum's low bits are the floor
  // q + kQBits as bits: the conversion is the addition of 1.5 * 2^23. The 64 keeps a q of -24 positive: next to a bucket's
  // border near 2048 a step count can round up by 2^-14 (8 of q) and c_low add a lack of 2^-13 (16).
  static constexpr float kRound = 12582912.0f + 64.0f;
  static constexpr unsigned kQBits = 0x4b400000u + 64u;
  // 2^23 (1 - exp(-f / 64)) = k1 f + k2 f^2 + k3 f^3 + k4 f^4, the next term below 2^-36 of it
  static constexpr float k1 = 131072.0f, k2 = -1024.0f, k3 = 16.0f / 3.0f, k4 = -1.0f / 48.0f;

  __device__ __forceinline__ float steps(float x) const { return (top - x) * c; }
  static __device__ __forceinline__ bool counts(float steps) { return steps < (float)kBuckets; }  // false for NaN
  // the bucket, or -1 for a weight that counts as 0
  __device__ __forceinline__ int bucket(float x) const {
    const float t = steps(x);
    return counts(t) ? (int)t : -1;
  }
  __device__ __forceinline__ unsigned part_bits(float x, float b) const {
    const float d = top - x, f = fmaf(d, c_low, fmaf(d, c, -b));
    return __float_as_uint(fmaf(f, fmaf(f, fmaf(f, fmaf(f, k4, k3), k2), k1), kRound));
  }
  // The same for two logits: bucket (in the low bits of `up`) and q. The steps are rounded before the floor is taken, as
  // `bucket` does it: a product that ran into the addition would put some logits into another bucket than the one they
  // are listed from. nz = f2_negzero() keeps it apart.
  __device__ __forceinline__ void two(float x, float y, F2 nz, float2& steps, float2& up, float2& q) const {
    const F2 minus = f2(-1.0f, -1.0f), tops = f2(top, top), cs = f2(c, c);
    const F2 d = fma2(f2(x, y), minus, tops), t = mul2(d, cs, nz), u = add2_down(t, f2(kFloor, kFloor));
    F2 f = fma2(u, minus, f2(kFloor, kFloor));  // - floor
    f = fma2(d, f2(c_low, c_low), fma2(d, cs, f));
    F2 e = fma2(f, f2(k4, k4), f2(k3, k3));
    e = fma2(f, e, f2(k2, k2));
    e = fma2(f, e, f2(k1, k1));
    e = fma2(f, e, f2(kRound, kRound));
    q = make_float2(f2_lo(e), f2_hi(e));
    steps = make_float2(f2_lo(t), f2_hi(t));
    up = make_float2(f2_lo(u), f2_hi(u));
  }
  // the weight in 64 bits, as the sums have it
  __device__ double weight(float x) const {
    const int b = bucket(x);
    return b < 0 ? 0.0
                 : exp(-(double)b / 64.0) * (double)(8388608 - (int)(part_bits(x, (float)b) - kQBits)) * (1.0 / 8388608.0);
  }
};

// What the leader asks of every CTA.
enum Op { kDone, kGather, kHistogram, kCountLeast };
constexpr int kRanges = 4;
struct Command {
  int op, first, last;  // buckets
  int bits;             // of the order that are fixed
  u64 prefix;           // their value
  // kGather, with more than one range: of first .. last only the buckets in these (closed)
  int ranges, from[kRanges], to[kRanges];
};

// The first of places 0 .. n - 1 that satisfies a condition which stays true from there on, n - 1 if none does: 32 places
// at a time. Every warp that takes part finds the same.
template <typename F>
__device__ __forceinline__ int first_of(int n, F holds) {
  const int lane = threadIdx.x % 32;
  int from = 0, left = n;
  while (left > 1) {
    const int step = (left + 31) / 32, end = min((lane + 1) * step, left);  // this lane's last place, from 1
    const unsigned hit = __ballot_sync(0xffffffffu, holds(from + end - 1));
    const int first = hit ? __ffs(hit) - 1 : 31;
    const int next = min(first * step, left - 1);
    left = min(step, left - next);
    from += next;
  }
  return from;
}

struct Sums {
  unsigned count[kBuckets];
  u64 q[kBuckets];  // signed sums
};
// Running sums up to and with each bucket.
struct Running {
  unsigned count[kBuckets];
  double mass[kBuckets];
  // the first bucket at which the count or the mass suffices (one with tokens in it), the last one if none does
  __device__ int find_count(unsigned k) const {
    return first_of(kBuckets, [&](int b) { return count[b] >= k; });
  }
  __device__ int find_mass(double want, bool more) const {
    const int b = first_of(kBuckets, [&](int i) { return more ? mass[i] > want : mass[i] >= want; });
    if (count[b] > before(b)) return b;
    // none does, or one without tokens: threads add up the running sums in orders of their own, so that they may rise by a
    // rounding there. The next one with tokens.
    return find_count(min(before(b) + 1, count[kBuckets - 1]));
  }
  __device__ unsigned before(int b) const { return b ? count[b - 1] : 0; }
  __device__ double mass_before(int b) const { return b ? mass[b - 1] : 0.0; }
};

struct Shared {
  union {
    unsigned hist[2][kBuckets];  // counts, sums of q + kQBits modulo 2^32
    struct {
      u64 list[kList];
      double prefix[kList];
    };
  };
  Sums sums;       // this CTA's
  union {
    Sums total;    // the leader's: of all CTAs
    Running bins;  // then over the bins of a crowded bucket, best first
  };
  Running row;     // the leader's: over the buckets
  u64 best[kMaxCluster];
  Command command;
  int listed, counted;
  u64 warp_best[kWarps];
  double warp_mass[kWarps];
  unsigned warp_count[kWarps];
};

// What is kept so far: everything before a bucket, and the first tokens of the bucket itself.
struct Cut {
  int bucket;
  unsigned count;
  double mass;  // of all that
};

template <int kType, int kCl>
struct Row {
  using V = TypeOf<kType>;
  using T = typename V::T;
  Shared& sh;
  const T* x;  // this CTA's logits
  int lo, n;   // the first one's index, their number
  Scale scale;
  bool top_infinite;
  float least, temperature;

  __device__ explicit Row(Shared& s) : sh(s) {}

  __device__ __forceinline__ void sync_all() {
    if (kCl > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename P>
  __device__ __forceinline__ P* at_rank(P* p, int r) {
    if (kCl > 1) return cg::this_cluster().map_shared_rank(p, r);
    return p;
  }

  // f(values, number of them, place of the first) for places from .. to - 1 of this CTA's logits: 16-byte loads, a few
  // at a time, between the first and the last aligned place, single ones outside.
  template <int kMany, typename F>
  __device__ __forceinline__ void for_each(int from, int to, F f) {
    constexpr int kVec = V::kVec;
    const int head = min(to - from, (int)((16 - reinterpret_cast<uintptr_t>(x + from) % 16) % 16 / sizeof(T)));
    const int vecs = (to - from - head) / kVec, tail = from + head + vecs * kVec;
    if ((int)threadIdx.x < head + (to - tail)) {
      const int at = (int)threadIdx.x < head ? from + (int)threadIdx.x : tail + (int)threadIdx.x - head;
      const float e[1] = {V::one(x + at)};
      f(e, at);
    }
    const uint4* v = reinterpret_cast<const uint4*>(x + from + head) + threadIdx.x;
    int at = from + head + (int)threadIdx.x * kVec, left = vecs - (int)threadIdx.x;
    for (; left > (kMany - 1) * kThreads; left -= kMany * kThreads) {
      uint4 b[kMany];
#pragma unroll
      for (int k = 0; k < kMany; ++k) b[k] = __ldg(v + k * kThreads);
#pragma unroll
      for (int k = 0; k < kMany; ++k) {
        float e[kVec];
        V::unpack(b[k], e);
        f(e, at + k * kThreads * kVec);
      }
      v += kMany * kThreads;
      at += kMany * kThreads * kVec;
    }
    for (; left > 0; left -= kThreads) {
      float e[kVec];
      V::unpack(__ldg(v), e);
      f(e, at);
      v += kThreads;
      at += kThreads * kVec;
    }
  }
  // a logit as the sums see it: where the largest is +infinity, one of 0 and nothing beside it
  __device__ __forceinline__ float seen(float v) const { return top_infinite ? (v == INFINITY ? 0.0f : -INFINITY) : v; }

  // ---- work of every CTA
  __device__ void clear_histogram() {
    for (int i = threadIdx.x; i < 2 * kBuckets; i += kThreads) sh.hist[0][i] = 0;
    __syncthreads();
  }
  static __device__ __forceinline__ void count_one(unsigned address, unsigned q) {
    asm volatile("red.shared.add.u32 [%0], 1;" ::"r"(address) : "memory");
    asm volatile("red.shared.add.u32 [%0 + %2], %1;" ::"r"(address), "r"(q), "n"(kBuckets * 4) : "memory");
  }
  // Counts and q of every bucket, or of the bins of one bucket, into sh.sums.
  template <bool kBins>
  __device__ void add_up(const Command& cmd) {
    unsigned c[kPerThread] = {};
    u64 q[kPerThread] = {};
    const int shift = kOrderBits - cmd.bits, digit = min(kDigit, shift);
    const int first = threadIdx.x * kPerThread;
    const F2 nz = f2_negzero();
    const unsigned hist = (unsigned)__cvta_generic_to_shared(&sh.hist[0][0]) - 4 * __float_as_uint(Scale::kFloor);
    for (int from = 0; from < max(n, 1); from += kFold) {
      clear_histogram();
      for_each<kAhead>(from, min(n, from + kFold), [&](const auto& e, int at) {
        constexpr int kN = (int)(sizeof(e) / sizeof(float));
        float v[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = e[i];
        if (top_infinite) {
#pragma unroll
          for (int i = 0; i < kN; ++i) v[i] = seen(v[i]);
        }
        if (kBins || kN == 1) {
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const int b = scale.bucket(v[i]);
            if (b < 0) continue;
            int bin = b;
            if (kBins) {
              const u64 o = order_of(v[i] + 0.0f, lo + at + i);
              if (b != cmd.first || (cmd.bits && o >> shift != cmd.prefix)) continue;
              bin = (int)(o >> (shift - digit)) & ((1 << digit) - 1);
            }
            atomicAdd(&sh.hist[0][bin], 1u);
            atomicAdd(&sh.hist[1][bin], scale.part_bits(v[i], (float)b));
          }
        } else {
#pragma unroll
          for (int i = 0; i + 1 < kN; i += 2) {
            float2 t, up, q;
            scale.two(v[i], v[i + 1], nz, t, up, q);
            // 4 * (bits of up) is 4 * bucket and a constant that goes into the address
            const unsigned a0 = hist + 4 * __float_as_uint(up.x), a1 = hist + 4 * __float_as_uint(up.y);
            if (Scale::counts(t.x)) count_one(a0, __float_as_uint(q.x));
            if (Scale::counts(t.y)) count_one(a1, __float_as_uint(q.y));
          }
        }
      });
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        const unsigned k = sh.hist[0][first + i];
        c[i] += k;
        // modulo 2^32 the sum of q + 64, which is positive and below 2^32
        q[i] += (u64)(sh.hist[1][first + i] - k * (Scale::kQBits - 64u)) - 64ull * k;
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      sh.sums.count[first + i] = c[i];
      sh.sums.q[first + i] = q[i];
    }
  }
  // Appends the tokens of the command's buckets to the leader's list. kMany: of several ranges of buckets.
  template <bool kMany>
  __device__ __forceinline__ void gather() {
    const Command& cmd = sh.command;
    int* const listed = at_rank(&sh.listed, 0);
    u64* const to = at_rank(sh.list, 0);
    const int shift = kOrderBits - cmd.bits, first_index = lo;
    const bool narrowed = cmd.bits > 0, infinite = top_infinite;
    const u64 prefix = cmd.prefix;
    const Scale sc = scale;
    auto append = [&](float v, int i) {
      const u64 o = order_of(v + 0.0f, first_index + i);
      if (narrowed && o >> shift != prefix) return;
      const int place = atomicAdd(listed, 1);
      if (place < kList) to[place] = o;
    };
    if (kMany) {
      float from[kRanges], end[kRanges];
#pragma unroll
      for (int k = 0; k < kRanges; ++k) {
        from[k] = k < cmd.ranges ? (float)cmd.from[k] : 1.0f;
        end[k] = k < cmd.ranges ? (float)(cmd.to[k] + 1) : 0.0f;
      }
      for_each<kAhead>(0, n, [&](const auto& e, int at) {
        constexpr int kN = (int)(sizeof(e) / sizeof(float));
        unsigned in = 0;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const float t = sc.steps(infinite ? seen(e[i]) : e[i]);
          bool one = false;
#pragma unroll
          for (int k = 0; k < kRanges; ++k) one = one || (t >= from[k] && t < end[k]);
          in |= one ? 1u << i : 0u;
        }
        if (in == 0) return;
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (in >> i & 1) append(seen(e[i]), at + i);
      });
    } else {
      // An interval that holds the logits of the buckets, a little wider: two comparisons settle almost every logit.
      const float from = (float)cmd.first, end = (float)(cmd.last + 1);
      const float a = sc.top - end / sc.c, b = sc.top - from / sc.c;
      const float wide = (fabsf(sc.top) + fmaxf(fabsf(a), fabsf(b))) * 1e-6f;
      const float v_low = a - wide, v_high = b + wide;  // NaN or infinite: every logit is looked at
      for_each<kAhead>(0, n, [&](const auto& e, int at) {
        constexpr int kN = (int)(sizeof(e) / sizeof(float));
        bool any = infinite;
#pragma unroll
        for (int i = 0; i < kN; ++i) any = any || !(e[i] < v_low || e[i] > v_high);
        if (!any) return;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const float v = seen(e[i]), t = sc.steps(v);
          if (t >= from && t < end) append(v, at + i);
        }
      });
    }
  }
  __device__ bool reaches_least(float v) const {
    return exp(((double)v - (double)scale.top) / (double)temperature) >= (double)least || v == scale.top;
  }
  __device__ __forceinline__ void count_least() {
    const Command& cmd = sh.command;
    int* counted = at_rank(&sh.counted, 0);
    for_each<1>(0, n, [&](const auto& e, int) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(e) / sizeof(float)); ++i) {
        const float v = seen(e[i]);
        const int b = scale.bucket(v);
        if (b >= cmd.first && b <= cmd.last && reaches_least(v)) atomicAdd(counted, 1);
      }
    });
  }
  // What the command asks for; not inlined, so that its loops have the registers to themselves.
  __device__ __noinline__ void serve() {
    const Command& cmd = sh.command;
    if (cmd.op == kGather) {
      if (cmd.ranges > 1) gather<true>();
      else gather<false>();
    } else if (cmd.op == kCountLeast) {
      count_least();
    } else if (cmd.op == kHistogram) {
      add_up<true>(cmd);
      share_sums();
    }
  }

  // ---- the leader's; every thread of it takes the same way
  __device__ void ask(const Command& cmd) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = sh.counted = 0;
    if (threadIdx.x < kCl) *at_rank(&sh.command, threadIdx.x) = cmd;
    sync_all();
    if (cmd.op == kDone) return;
    serve();
    sync_all();
  }

  // The CTAs' sums into the leader's: each adds an eighth of the buckets over all of them. Ends with all CTAs in step.
  __device__ void share_sums() {
    sync_all();
    if (kCl == 1) return;
    constexpr int kEach = kBuckets / kCl, kLanes = kThreads / kEach;  // threads per bucket
    constexpr int kTurns = kLanes ? 1 : kEach / kThreads, kSplit = kLanes ? kLanes : 1;
    const int rank = (int)cg::this_cluster().block_rank();
#pragma unroll
    for (int turn = 0; turn < kTurns; ++turn) {
      const int b = rank * kEach + turn * kThreads + (int)threadIdx.x / kSplit, part = threadIdx.x % kSplit;
      unsigned c = 0;
      u64 q = 0;
#pragma unroll
      for (int r = 0; r < kCl / kSplit; ++r) {
        const Sums* s = at_rank(&sh.sums, r * kSplit + part);
        c += s->count[b];
        q += s->q[b];
      }
#pragma unroll
      for (int i = 1; i < kSplit; i <<= 1) {
        c += __shfl_xor_sync(0xffffffffu, c, i);
        q += __shfl_xor_sync(0xffffffffu, q, i);
      }
      if (part == 0) {
        at_rank(&sh.total, 0)->count[b] = c;
        at_rank(&sh.total, 0)->q[b] = q;
      }
    }
    sync_all();
  }
  // The running sums of all CTAs. base < 0: over the buckets; else over the bins of bucket `base`, the largest first.
  __device__ void run_sums(Running& to, int base) {
    static_assert(kPerThread == 4, "16 bytes a thread");
    const int first = threadIdx.x * kPerThread;
    const int from = base < 0 ? first : kBuckets - kPerThread - first;
    const Sums& s = kCl == 1 ? sh.sums : sh.total;
    unsigned c[kPerThread];
    u64 q[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      c[i] = s.count[from + (base < 0 ? i : kPerThread - 1 - i)];
      q[i] = s.q[from + (base < 0 ? i : kPerThread - 1 - i)];
    }
    double e = exp(-(double)(base < 0 ? first : base) / 64.0) * (1.0 / 8388608.0), m[kPerThread];
    unsigned tc = 0;
    double tm = 0.0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      tc = c[i] += tc;
      tm = m[i] = tm + e * (double)(long long)(((u64)(c[i] - (i ? c[i - 1] : 0)) << 23) - q[i]);
      if (base < 0) e *= 0.98449643700540841;  // exp(-1 / 64)
    }
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    unsigned sc = tc;
    double sm = tm;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const unsigned vc = __shfl_up_sync(0xffffffffu, sc, i);
      const double vm = __shfl_up_sync(0xffffffffu, sm, i);
      if (lane >= i) {
        sc += vc;
        sm += vm;
      }
    }
    if (lane == 31) {
      sh.warp_count[warp] = sc;
      sh.warp_mass[warp] = sm;
    }
    sc = __shfl_up_sync(0xffffffffu, sc, 1);
    sm = __shfl_up_sync(0xffffffffu, sm, 1);
    if (lane == 0) sc = 0, sm = 0.0;
    __syncthreads();
    unsigned wc = 0;
    double wm = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warp) {
        wc += sh.warp_count[w];
        wm += sh.warp_mass[w];
      }
    // every thread has read its sums by now: `to` may lie over them
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      to.count[first + i] = wc + sc + c[i];
      to.mass[first + i] = wm + (sm + m[i]);
    }
    __syncthreads();
  }

  // Sorts the gathered tokens, best first, and sums their weights: prefix[i] = sum of weights 0 .. i.
  __device__ void sort_list(int n_list) {
    u64* list = sh.list;
    int size = 2;
    while (size < n_list) size <<= 1;
    for (int i = n_list + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    // a warp's turn covers 64 neighbours: steps within them need only their own warp
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (j >= 32 || j == k >> 1) __syncthreads();
        else __syncwarp();
        for (int t = threadIdx.x; t < size / 2; t += kThreads) {
          const int i = 2 * t - (t & (j - 1)), p = i + j;
          const u64 u = list[i], v = list[p];
          if ((u < v) == ((i & k) == 0)) {
            list[i] = v;
            list[p] = u;
          }
        }
      }
    __syncthreads();
    constexpr int kEach = kList / kThreads;
    const int each = (n_list + kThreads - 1) / kThreads, i0 = each * threadIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    double w[kEach], own = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (i < each && i0 + i < n_list) own += scale.weight(value_of(list[i0 + i]));
      w[i] = own;
    }
    double s = own;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, s, i);
      if (lane >= i) s += v;
    }
    if (lane == 31) sh.warp_mass[warp] = s;
    s = __shfl_up_sync(0xffffffffu, s, 1);
    if (lane == 0) s = 0.0;
    __syncthreads();
    double before = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i)
      if (i < warp) before += sh.warp_mass[i];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < each && i0 + i < n_list) sh.prefix[i0 + i] = before + (s + w[i]);
    __syncthreads();
  }
  // A mass inside bucket b, kept from leaving it by the rounding of its sum.
  __device__ double within(int b, double m) const { return fmin(fmax(m, sh.row.mass_before(b)), sh.row.mass[b]); }
  // Inside bucket b: the cut at the first token with at least `need` tokens of the bucket up to it (need > 0), or a mass
  // of everything up to it that reaches (more: exceeds) want; at most `most` tokens. Also that token. `listed`: the length
  // of the sorted list, which holds whole buckets; 0 as soon as a bucket had to be gathered by itself.
  __device__ Cut resolve(int b, unsigned need, double want, bool more, unsigned most, int& listed, u64& order) {
    const int from = first_of(listed, [&](int i) { return scale.bucket(value_of(sh.list[i])) >= b; });
    // a rounding may have moved a border into a bucket that is not in the list
    if (listed && scale.bucket(value_of(sh.list[from])) != b) listed = 0;
    if (listed) {
      const unsigned n_in = sh.row.count[b] - sh.row.before(b);
      const double m0 = sh.row.mass_before(b) - (from ? sh.prefix[from - 1] : 0.0);
      const int at = first_of((int)min(min(most, n_in), (unsigned)(listed - from)), [&](int i) {
        const double m = m0 + sh.prefix[from + i];
        return need ? (unsigned)i + 1 >= need : (more ? m > want : m >= want);
      });
      order = sh.list[from + at];
      return {b, (unsigned)at + 1, within(b, m0 + sh.prefix[from + at])};
    }
    Command cmd{kGather, b, b, 0, 0, 0, {}, {}};
    unsigned c0 = 0, n_in = sh.row.count[b] - sh.row.before(b);
    double m0 = sh.row.mass_before(b);
    most = min(most, n_in);
    while (n_in > kList) {  // crowded: narrow by digits of the order, from the top
      cmd.op = kHistogram;
      ask(cmd);
      run_sums(sh.bins, b);
      int bin = need ? sh.bins.find_count(need - c0) : sh.bins.find_mass(want - m0, more);
      bin = min(bin, sh.bins.find_count(most - c0));
      const int digit = min(kDigit, kOrderBits - cmd.bits);
      cmd.prefix = cmd.prefix << digit | (u64)(kBuckets - 1 - bin);
      cmd.bits += digit;
      n_in = sh.bins.count[bin] - sh.bins.before(bin);
      c0 += sh.bins.before(bin);
      m0 += sh.bins.mass_before(bin);
      cmd.op = kGather;
    }
    ask(cmd);
    sort_list((int)n_in);
    const int at = first_of(min(n_in, most - c0), [&](int i) {
      return need ? c0 + i + 1 >= need : (more ? m0 + sh.prefix[i] > want : m0 + sh.prefix[i] >= want);
    });
    order = sh.list[at];
    return {b, c0 + at + 1, within(b, m0 + sh.prefix[at])};
  }

  __device__ void lead(float u, int k, float p, u64 best, u64& order, double& total) {
    bool use_p = p < 1.0f, use_least = least > 0.0f;
    if ((use_p && p <= 0.0f) || least > 1.0f) k = 1;
    if (k == 1) {
      order = best;
      total = 1.0;
      return;
    }
    run_sums(sh.row, -1);
    const Running& row = sh.row;
    const unsigned all = row.count[kBuckets - 1];
    if (k < 0 || (unsigned)k >= all) k = 0;
    // Where min_p's border lies: tokens of these buckets are compared in 64 bits. A logit's own step count is rounded to
    // fp32, so next to a bucket's border the neighbour is looked at too.
    int least_from = kBuckets, least_to = kBuckets;
    if (use_least) {
      const double z = -log((double)least) * 64.0;
      use_least = z < kBuckets;
      if (use_least) {
        least_from = max(0, (int)(z - 1.0 / 512.0));
        least_to = min(kBuckets - 1, max(0, (int)(z + 1.0 / 512.0)));
      }
    }
    const double draw = u > 0.0f ? fmin((double)u, 1.0) : 0.0;  // from 1 on: the last one kept

    // The buckets that borders and draw may fall in, from the sums alone: a border inside a bucket leaves the mass up to
    // it between that before and that behind the bucket, and so what depends on it between two buckets. Mostly they
    // hold few tokens, which are gathered and sorted at once.
    const double whole = row.mass[kBuckets - 1];
    Command cmd{kGather, kBuckets, 0, 0, 0, 0, {}, {}};
    unsigned listed = 0;
    auto want_range = [&](int from, int to) {
      from = min(from, to);  // a draw of all that is kept is sought behind it
      cmd.from[cmd.ranges] = from;
      cmd.to[cmd.ranges++] = to;
      cmd.first = min(cmd.first, from);
      cmd.last = max(cmd.last, to);
      listed += row.count[to] - row.before(from);
    };
    double low = whole, high = whole;  // of the mass that is kept
    int cut_to = kBuckets - 1;         // no kept token lies behind
    if (k) {
      cut_to = row.find_count(k);
      low = row.mass_before(cut_to);
      high = row.mass[cut_to];
      if (row.count[cut_to] == (unsigned)k) low = high;
      else want_range(cut_to, cut_to);
    }
    if (use_p) {
      const int from = row.find_mass((double)p * low, false), to = min(cut_to, row.find_mass((double)p * high, false));
      want_range(from, to);
      low = row.mass_before(from);
      high = row.mass[to];
      cut_to = to;
    }
    if (use_least && least_from <= cut_to) {
      if (row.count[least_to] > row.before(least_from)) want_range(least_from, least_to);
      low = fmin(low, row.mass_before(least_from));
      high = fmin(high, row.mass[least_to]);
    }
    want_range(row.find_mass(draw * low, true), min(cut_to, row.find_mass(draw * high, true)));
    int n_list = 0;
    if (listed <= kList) {
      ask(cmd);
      n_list = sh.listed <= kList ? sh.listed : 0;  // the list's bounds do not rest on the sums
      sort_list(n_list);
    }

    Cut cut{kBuckets, 0, row.mass[kBuckets - 1]};  // nothing is cut off
    if (k) {
      const int b = row.find_count(k);
      if (row.count[b] == (unsigned)k) cut = {b, (unsigned)k - row.before(b), row.mass[b]};
      else cut = resolve(b, (unsigned)k - row.before(b), 0.0, false, ~0u, n_list, order);
    }
    if (use_p) {
      const double want = (double)p * cut.mass;
      const int b = row.find_mass(want, false);
      if (b < cut.bucket || (b == cut.bucket && cut.count > 0)) cut = resolve(b, 0, want, false, b < cut.bucket ? ~0u : cut.count, n_list, order);
    }
    if (use_least && least_from <= cut.bucket) {
      const unsigned has = row.count[least_to] - row.before(least_from);
      unsigned in = 0;
      if (n_list) {
        if (has) {
          const int from = first_of(n_list, [&](int i) { return scale.bucket(value_of(sh.list[i])) >= least_from; });
          in = first_of((int)has + 1, [&](int i) { return i == (int)has || !reaches_least(value_of(sh.list[from + i])); });
        }
      } else {
        ask({kCountLeast, least_from, least_to, 0, 0, 0, {}, {}});
        in = (unsigned)sh.counted;
      }
      const unsigned reach = row.before(least_from) + in;  // at least 1: the best one
      if (cut.bucket == kBuckets || reach < row.before(cut.bucket) + cut.count) {
        const int b = row.find_count(reach);
        if (row.count[b] == reach) cut = {b, reach - row.before(b), row.mass[b]};
        else cut = resolve(b, reach - row.before(b), 0.0, false, ~0u, n_list, order);
      }
    }
    total = cut.mass;
    const double want = draw * total;
    int b = row.find_mass(want, true);
    if (b < cut.bucket || (b == cut.bucket && cut.count > 0)) {
      resolve(b, 0, want, true, b < cut.bucket ? ~0u : cut.count, n_list, order);
    } else {  // the draw fell behind the cut by a rounding: the last one kept
      const unsigned kept = row.before(cut.bucket) + cut.count;
      b = row.find_count(kept);
      resolve(b, kept - row.before(b), 0.0, false, ~0u, n_list, order);
    }
  }
};

// A cluster of 8 has its SMs to itself and takes the registers that the leader's part wants (1 row: 19.2 us, 21.5 with 64).
template <int kType, int kCl>
__global__ void __cluster_dims__(kCl, 1, 1) __launch_bounds__(kThreads, kCl == kMaxCluster ? 1 : 2)
    sample_kernel(Sample a, int slice) {
  using R = Row<kType, kCl>;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  const int row = blockIdx.x / kCl, rank = blockIdx.x % kCl, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  R r(sh);
  // another CTA's shared memory may be written once that CTA has started: each says so here, and waits below
  if (kCl > 1) cg::this_cluster().barrier_arrive();
  r.lo = min(a.vocab, rank * slice);
  r.n = min(slice, a.vocab - r.lo);
  r.x = static_cast<const typename R::T*>(a.logits) + (long long)row * a.stride + r.lo;

  float top = -INFINITY;
  int top_at = 0;
  r.template for_each<kAhead>(0, r.n, [&](const auto& e, int at) {
    float m = e[0];
#pragma unroll
    for (int i = 1; i < (int)(sizeof(e) / sizeof(float)); ++i) m = fmaxf(m, e[i]);
    if (m > top || (m == top && at < top_at)) {  // never for NaN
      top = m;
      top_at = at;
    }
  });
  // the place of the group's first such value
  while (top > -INFINITY && R::V::one(r.x + top_at) != top) ++top_at;
  u64 best = top > -INFINITY ? order_of(top + 0.0f, r.lo + top_at) : 0;  // -0 becomes +0: they tie
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, s));
  if (lane == 0) sh.warp_best[warp] = best;
  __syncthreads();
  if (kCl > 1) cg::this_cluster().barrier_wait();
  if (threadIdx.x < kCl) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) best = max(best, sh.warp_best[w]);
    r.at_rank(sh.best, threadIdx.x)[rank] = best;
  }
  r.sync_all();
  best = 0;
#pragma unroll
  for (int c = 0; c < kCl; ++c) best = max(best, sh.best[c]);

  const float t = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  if (best == 0 || !(t >= 1.17549435e-38f)) {
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = best == 0 ? -1 : index_of(best);
      if (a.probs) a.probs[row] = best == 0 ? 0.0f : 1.0f;
    }
    return;
  }
  r.top_infinite = value_of(best) == INFINITY;
  r.temperature = fmaxf(t, 3.7615819e-37f);  // 2^-121: 64 / t stays finite, so that the best token stays at 0 steps
  r.scale = Scale(r.seen(value_of(best)), r.temperature);
  r.least = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  r.template add_up<false>({kHistogram, 0, kBuckets - 1, 0, 0, 0, {}, {}});
  r.share_sums();
  if (rank == 0) {
    u64 order = best;
    double total = 1.0;
    r.lead(__ldg(a.uniforms + row), a.top_k ? __ldg(a.top_k + row) : 0, a.top_p ? __ldg(a.top_p + row) : 1.0f, best, order, total);
    if (threadIdx.x == 0) {
      a.tokens[row] = index_of(order);
      // the best token may be +infinity, which the sums see as 0; its weight is 1 in any case
      if (a.probs) a.probs[row] = order == best ? (float)(1.0 / total) : (float)(r.scale.weight(value_of(order)) / total);
    }
    if (kCl > 1) r.ask({kDone, 0, 0, 0, 0, 0, {}, {}});
  } else {
    for (;;) {
      r.sync_all();
      if (sh.command.op == kDone) break;
      r.serve();
      r.sync_all();
    }
  }
}

template <int kType, int kCl>
cudaError_t launch(const Sample& a, cudaStream_t s) {
  const int slice = ((a.vocab + kCl - 1) / kCl + 15) / 16 * 16;
  const cudaError_t e = cudaFuncSetAttribute(sample_kernel<kType, kCl>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
  if (e != cudaSuccess) return e;
  sample_kernel<kType, kCl><<<(unsigned)a.rows * kCl, kThreads, sizeof(Shared), s>>>(a, slice);
  return cudaGetLastError();
}

template <int kType>
cudaError_t launch(const Sample& a, cudaStream_t s) {
  const long long rows = a.rows;
  if (a.vocab <= kOneCta || rows * 2 > 2 * kSms) return launch<kType, 1>(a, s);
  if (rows * 4 > 2 * kSms) return launch<kType, 2>(a, s);
  return rows * 8 > kSms ? launch<kType, 4>(a, s) : launch<kType, 8>(a, s);
}

}  // namespace

cudaError_t launch_sample(const Sample& a, int type, cudaStream_t s) {
  return type == 0 ? launch<0>(a, s) : type == 1 ? launch<1>(a, s) : launch<2>(a, s);
}

}  // namespace sampling
}  // namespace qb
