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
// tokens of such buckets are gathered and sorted. A weight is off by at most 2^-24 of its bucket's largest (the
// rounding of q; f is exact to 2^-30).
//
// One cluster of 8 CTAs takes a row, an eighth of the logits each, in shared memory: they are read from HBM once. Small
// vocabularies take one CTA. The first CTA leads: it reads the others' bucket sums through distributed shared
// memory, decides, and asks for what it needs to see. Bound: the latency of those steps for few rows (8 SMs of 148
// work on a row), bytes for many.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "sample.h"

namespace cg = cooperative_groups;

namespace qb {
namespace sampling {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBuckets = 2048;
constexpr int kPerThread = kBuckets / kThreads;
constexpr int kList = 1024;  // tokens that are sorted at once
constexpr int kOrderBits = 50;
constexpr int kDigit = 11;   // bits by which a crowded bucket is narrowed at a time
constexpr int kCluster = 8;
constexpr int kOneCta = 8192;  // vocabularies up to this size take one CTA: less to read than a cluster costs to sync

typedef unsigned long long u64;

template <int kType>
struct TypeOf;
template <>
struct TypeOf<0> {
  using T = float;
};
template <>
struct TypeOf<1> {
  using T = __half;
};
template <>
struct TypeOf<2> {
  using T = __nv_bfloat16;
};
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

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

// z = (top - x) / temperature in parts: bucket and q. The product with 1 / temperature = c + c_low is exact to
// about 2^-48, and so is its distance to the bucket's border.
struct Scale {
  float top, c, c_low;
  __device__ Scale(float top_, float t) : top(top_), c(1.0f / t) {
    c_low = c > 0.0f ? fmaf(-t, c, 1.0f) * c : 0.0f;
    if (!(fabsf(c_low) < c)) c_low = 0.0f;
  }
  // the bucket, or -1 for a weight that counts as 0
  __device__ __forceinline__ int bucket(float x, float& d) const {
    d = x == top ? 0.0f : top - x;  // +infinity ties with itself
    const float t = d * c * 64.0f;
    return t < (float)kBuckets ? (int)t : -1;
  }
  __device__ __forceinline__ int bucket(float x) const {
    float d;
    return bucket(x, d);
  }
  __device__ __forceinline__ int part(float x, float d, int b) const {
    const float s = d == 0.0f ? 0.0f : top - d;  // what x is short of top - d, exactly (two-sum)
    const float low = d == 0.0f ? 0.0f : (top - (s + d)) - (x - s);
    float f = fmaf(d, c, -(float)b * (1.0f / 64.0f)) + fmaf(d, c_low, low * c);
    f = fmaxf(f, 0.0f);
    // 1 - exp(-f) for f < 1/64: the series' next term, f^5 / 120, is below 2^-36
    const float e = f * fmaf(f, fmaf(f, fmaf(f, -1.0f / 24.0f, 1.0f / 6.0f), -0.5f), 1.0f);
    return min(__float2int_rn(e * 8388608.0f), 131071);
  }
  // the weight in 64 bits, as the sums have it
  __device__ double weight(float x) const {
    float d;
    const int b = bucket(x, d);
    return b < 0 ? 0.0 : exp(-(double)b / 64.0) * (double)(8388608 - part(x, d, b)) * (1.0 / 8388608.0);
  }
};

// What the leader asks of every CTA.
enum Op { kDone, kGather, kHistogram, kCountLeast };
struct Command {
  int op, first, last;  // buckets
  int bits;             // of the order that are fixed
  u64 prefix;           // their value
};

struct Shared {
  u64 best[kCluster];
  Command command;
  int listed, counted;
  u64 warp_best[kWarps];
  double warp_mass[kWarps];
  unsigned warp_count[kWarps];
  int found;
  double answer_mass;
  unsigned answer_count;
  double bucket_mass;
  unsigned bucket_count;
};

// A border or a draw inside one bucket, or the whole kept set: how many tokens up to and with the found one.
struct Cut {
  int bucket;
  unsigned count;  // tokens of the bucket that are kept
  double mass;     // of everything up to there
};

template <int kType, int kCl>
struct Row {
  using T = typename TypeOf<kType>::T;
  const Sample& a;
  Shared& sh;
  float* x;             // this CTA's logits; NaN as -infinity
  unsigned* hist;       // [2][kBuckets]: counts, sums of q
  u64* list;            // [kList], in the histogram's place
  double* prefix;       // [kList], behind it
  int rank, lo, n;
  Scale scale{0.0f, 1.0f};
  double least = 0.0, temperature = 1.0;
  // the leader's bucket sums, kPerThread buckets a thread
  unsigned count[kPerThread], count_before;
  double mass[kPerThread], mass_before;
  unsigned all_count;
  double all_mass;

  __device__ Row(const Sample& a_, Shared& s_) : a(a_), sh(s_) {}

  __device__ __forceinline__ void sync_all() {
    if (kCl > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename P>
  __device__ __forceinline__ P* at_rank(P* p, int r) {
    if (kCl > 1) return cg::this_cluster().map_shared_rank(p, r);
    return p;
  }

  // ---- work of every CTA
  __device__ void add_up(const Command& cmd) {
    const int shift = kOrderBits - cmd.bits, digit = min(kDigit, shift);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      if (!(v > -INFINITY)) continue;
      float d;
      const int b = scale.bucket(v, d);
      if (b < cmd.first || b > cmd.last) continue;
      const u64 o = order_of(v, lo + i);
      if (cmd.bits && o >> shift != cmd.prefix) continue;
      const int bin = cmd.first == cmd.last ? (int)(o >> (shift - digit)) & ((1 << digit) - 1) : b;
      atomicAdd(hist + bin, 1u);
      atomicAdd(hist + kBuckets + bin, (unsigned)scale.part(v, d, b));
    }
  }
  __device__ void clear_histogram() {
    for (int i = threadIdx.x; i < 2 * kBuckets; i += kThreads) hist[i] = 0;
    __syncthreads();
  }
  __device__ void gather(const Command& cmd) {
    int* listed = at_rank(&sh.listed, 0);
    u64* to = at_rank(list, 0);
    const int shift = kOrderBits - cmd.bits;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      if (!(v > -INFINITY)) continue;
      const int b = scale.bucket(v);
      if (b < cmd.first || b > cmd.last) continue;
      const u64 o = order_of(v, lo + i);
      if (cmd.bits && o >> shift != cmd.prefix) continue;
      const int at = atomicAdd(listed, 1);
      if (at < kList) to[at] = o;
    }
  }
  __device__ bool reaches_least(float v) const {
    return exp(((double)v - (double)scale.top) / temperature) >= least || v == scale.top;
  }
  __device__ void count_least(const Command& cmd) {
    int* counted = at_rank(&sh.counted, 0);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float v = x[i];
      if (v > -INFINITY && scale.bucket(v) == cmd.first && reaches_least(v)) atomicAdd(counted, 1);
    }
  }
  __device__ void serve(const Command& cmd) {
    if (cmd.op == kGather) gather(cmd);
    else if (cmd.op == kCountLeast) count_least(cmd);
    else if (cmd.op == kHistogram) {
      clear_histogram();
      add_up(cmd);
    }
  }

  // ---- the leader's
  __device__ void ask(const Command& cmd) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = sh.counted = 0;
    if (threadIdx.x < kCl) *at_rank(&sh.command, threadIdx.x) = cmd;
    sync_all();
    if (cmd.op == kDone) return;
    serve(cmd);
    sync_all();
  }

  // The CTAs' histograms as bucket sums. `base` < 0: buckets of z; else bins inside bucket `base`, largest first.
  __device__ void read_sums(int base, int bins) {
    unsigned c[kPerThread] = {};
    u64 q[kPerThread] = {};
    static_assert(kPerThread == 4, "16 bytes a thread");
    const int first = threadIdx.x * kPerThread;
    const int from = base < 0 ? first : kBuckets - kPerThread - first;
#pragma unroll
    for (int r = 0; r < kCl; ++r) {
      const unsigned* h = at_rank(hist, r);
      const uint4 n4 = *reinterpret_cast<const uint4*>(h + from), q4 = *reinterpret_cast<const uint4*>(h + kBuckets + from);
      const unsigned nn[4] = {n4.x, n4.y, n4.z, n4.w}, qq[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] += nn[base < 0 ? i : 3 - i];
        q[i] += qq[base < 0 ? i : 3 - i];
      }
    }
    unsigned tc = 0;
    double tm = 0.0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const double e = c[i] ? exp(-(double)(base < 0 ? first + i : base) / 64.0) : 0.0;
      count[i] = c[i];
      mass[i] = e * ((double)(((u64)c[i] << 23) - q[i]) * (1.0 / 8388608.0));
      tc += count[i];
      tm += mass[i];
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
    __syncthreads();
    if (lane == 31) {
      sh.warp_count[warp] = sc;
      sh.warp_mass[warp] = sm;
    }
    __syncthreads();
    count_before = sc - tc;
    mass_before = sm - tm;
    all_count = 0;
    all_mass = 0.0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        count_before += sh.warp_count[w];
        mass_before += sh.warp_mass[w];
      }
      all_count += sh.warp_count[w];
      all_mass += sh.warp_mass[w];
    }
  }

  struct Found {
    int bucket;
    unsigned count_before, count;
    double mass_before, mass;
  };
  // The first bucket that is not empty and satisfies reached(count up to its end, mass up to its end); the last one
  // that is not empty if none does.
  template <typename F>
  __device__ Found find(F reached) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = kBuckets;
    __syncthreads();
    unsigned c = count_before;
    double m = mass_before;
    int mine = kBuckets, last = -1;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      c += count[i];
      m += mass[i];
      if (count[i] == 0) continue;
      last = (int)threadIdx.x * kPerThread + i;
      if (mine == kBuckets && reached(c, m)) mine = last;
    }
    if (mine < kBuckets) atomicMin(&sh.found, mine);
    __syncthreads();
    if (sh.found == kBuckets) {  // none (a sum's rounding): uniform over the CTA
      __syncthreads();
      if (threadIdx.x == 0) sh.found = -1;
      __syncthreads();
      if (last >= 0) atomicMax(&sh.found, last);
      __syncthreads();
    }
    return at_bucket(sh.found);
  }
  __device__ Found at_bucket(int b) {
    __syncthreads();
    if ((int)threadIdx.x == b / kPerThread) {
      unsigned c = count_before;
      double m = mass_before;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        if (i == b % kPerThread) {
          sh.answer_count = c;
          sh.answer_mass = m;
          sh.bucket_count = count[i];
          sh.bucket_mass = mass[i];
        }
        c += count[i];
        m += mass[i];
      }
    }
    __syncthreads();
    return {b, sh.answer_count, sh.bucket_count, sh.answer_mass, sh.bucket_mass};
  }

  // Sorts the gathered tokens, best first, and sums their weights: prefix[i] = sum of weights 0 .. i.
  __device__ void sort_list(int n_list) {
    int size = 2;
    while (size < n_list) size <<= 1;
    __syncthreads();
    for (int i = n_list + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
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
    const int i0 = 2 * threadIdx.x;
    const double w0 = i0 < n_list ? scale.weight(value_of(list[i0])) : 0.0;
    const double w1 = i0 + 1 < n_list ? scale.weight(value_of(list[i0 + 1])) : 0.0;
    double s = w0 + w1;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, s, i);
      if (lane >= i) s += v;
    }
    if (lane == 31) sh.warp_mass[warp] = s;
    __syncthreads();
    for (int w = 0; w < warp; ++w) s += sh.warp_mass[w];
    if (i0 < kList) {
      prefix[i0] = s - w1;
      prefix[i0 + 1] = s;
    }
    __syncthreads();
  }
  // The first place of the sorted list that satisfies reached(its number from 1, the sum with it); the last if none does.
  template <typename F>
  __device__ int first_place(int n_list, F reached) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = n_list - 1;
    __syncthreads();
    for (int i = threadIdx.x; i < n_list; i += kThreads)
      if (reached((unsigned)i + 1, prefix[i])) {
        atomicMin(&sh.found, i);
        break;
      }
    __syncthreads();
    return sh.found;
  }

  // Inside bucket f: the first token for which reached(tokens, mass) holds, both counted from the bucket's first token.
  // Leaves the sorted neighbourhood in the list. Returns the cut at that token and the token.
  template <typename F>
  __device__ Cut resolve(const Found& f, F reached, u64& order) {
    Command cmd{kGather, f.bucket, f.bucket, 0, 0};
    unsigned c0 = 0, n_in = f.count;
    double m0 = 0.0;
    if (n_in > kList) {
      // crowded: narrow by digits of the order, from the top. The bucket sums make room for the bins' and return after.
      unsigned keep_c[kPerThread + 2];
      double keep_m[kPerThread + 2];
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        keep_c[i] = count[i];
        keep_m[i] = mass[i];
      }
      keep_c[kPerThread] = count_before;
      keep_m[kPerThread] = mass_before;
      keep_c[kPerThread + 1] = all_count;
      keep_m[kPerThread + 1] = all_mass;
      while (n_in > kList) {
        cmd.op = kHistogram;
        ask(cmd);
        read_sums(f.bucket, kBuckets);
        const Found bin = find([&](unsigned c, double m) { return reached(c0 + c, m0 + m); });
        const int digit = min(kDigit, kOrderBits - cmd.bits);
        cmd.prefix = cmd.prefix << digit | (u64)(kBuckets - 1 - bin.bucket);
        cmd.bits += digit;
        c0 += bin.count_before;
        m0 += bin.mass_before;
        n_in = bin.count;
      }
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        count[i] = keep_c[i];
        mass[i] = keep_m[i];
      }
      count_before = keep_c[kPerThread];
      mass_before = keep_m[kPerThread];
      all_count = keep_c[kPerThread + 1];
      all_mass = keep_m[kPerThread + 1];
      cmd.op = kGather;
    }
    ask(cmd);
    sort_list((int)n_in);
    const int at = first_place((int)n_in, [&](unsigned c, double m) { return reached(c0 + c, m0 + m); });
    order = list[at];
    const Cut cut{f.bucket, c0 + at + 1, f.mass_before + m0 + prefix[at]};
    __syncthreads();
    return cut;
  }

  __device__ void lead(float u, int k, float p, float mp, u64 best, u64& order, double& total) {
    read_sums(-1, kBuckets);
    bool use_p = p < 1.0f, use_least = mp > 0.0f;
    if ((use_p && p <= 0.0f) || mp > 1.0f) k = 1;
    if (k == 1) {
      order = best;
      total = 1.0;
      return;
    }
    if (k < 0 || (unsigned)k >= all_count) k = 0;
    int least_bucket = kBuckets;
    if (use_least) {
      least = mp;
      const double z = -log((double)mp) * 64.0;
      use_least = z < kBuckets;
      least_bucket = use_least ? max(0, (int)z) : kBuckets;
    }
    const double draw = u > 0.0f ? (double)u : 0.0;

    // a bucket that no kept token lies behind, and that the sums which decide do not reach behind: top_p after top_k
    // needs the sum of all that top_k keeps
    if (k || use_p || use_least) {
      int bound = kBuckets - 1;
      if (k) bound = find([&](unsigned c, double) { return c >= (unsigned)k; }).bucket;
      else if (use_p) bound = find([&](unsigned, double m) { return m >= (double)p * all_mass; }).bucket;
      if (use_least && !(k && use_p)) bound = min(bound, least_bucket);
      const Found f = at_bucket(bound);
      const unsigned n_in = f.count_before + f.count;
      if (n_in <= kList) {
        // few: sort them all and filter there
        ask({kGather, 0, bound, 0, 0});
        sort_list((int)n_in);
        int kept = k ? min(k, (int)n_in) : (int)n_in;
        if (use_p) {
          // without top_k the whole sum counts, behind the bound too
          const double want = (double)p * (k ? prefix[kept - 1] : all_mass);
          kept = min(kept, 1 + first_place((int)n_in, [&](unsigned, double m) { return m >= want; }));
        }
        if (use_least) {
          const int out = first_place((int)n_in, [&](unsigned c, double) { return !reaches_least(value_of(list[c - 1])); });
          if (!reaches_least(value_of(list[out]))) kept = min(kept, max(1, out));
        }
        total = prefix[kept - 1];
        const double want = draw * total;
        const int at = min(kept - 1, first_place((int)n_in, [&](unsigned, double m) { return m > want; }));
        order = list[at];
        return;
      }
    }

    Cut cut{kBuckets, 0, all_mass};  // nothing is cut off
    if (k) {
      const Found f = find([&](unsigned c, double) { return c >= (unsigned)k; });
      const unsigned in = (unsigned)k - f.count_before;
      if (in == f.count) cut = {f.bucket, in, f.mass_before + f.mass};
      else cut = resolve(f, [&](unsigned c, double) { return c >= in; }, order);
    }
    if (use_p) {
      const double want = (double)p * cut.mass;
      const Found f = find([&](unsigned, double m) { return m >= want; });
      if (f.bucket <= cut.bucket) {
        const Cut by_p = resolve(f, [&](unsigned, double m) { return f.mass_before + m >= want; }, order);
        if (f.bucket < cut.bucket || by_p.count < cut.count) cut = by_p;
      }
    }
    if (use_least && least_bucket <= cut.bucket) {
      const Found f = at_bucket(least_bucket);
      ask({kCountLeast, least_bucket, least_bucket, 0, 0});
      const unsigned in = (unsigned)sh.counted;
      if (least_bucket < cut.bucket || in < cut.count) {
        if (in == 0) cut = {least_bucket, 0, f.mass_before};
        else if (in == f.count) cut = {least_bucket, in, f.mass_before + f.mass};
        else cut = resolve(f, [&](unsigned c, double) { return c >= in; }, order);
      }
    }
    total = cut.mass;
    const double want = draw * total;
    const Found f = find([&](unsigned, double m) { return m > want; });
    if (f.bucket < cut.bucket || (f.bucket == cut.bucket && cut.count > 0)) {
      const unsigned most = f.bucket < cut.bucket ? f.count : cut.count;
      resolve(f, [&](unsigned c, double m) { return c >= most || f.mass_before + m > want; }, order);
    } else {  // the draw fell behind the cut by a rounding: the last one kept
      const unsigned kept = at_bucket(cut.bucket).count_before + cut.count;
      const Found g = find([&](unsigned c, double) { return c >= kept; });
      resolve(g, [&](unsigned c, double) { return g.count_before + c >= kept; }, order);
    }
  }
};

template <int kType, int kCl>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(Sample a, int slice) {
  using R = Row<kType, kCl>;
  using T = typename R::T;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  const int row = blockIdx.x / kCl, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  R r(a, sh);
  r.rank = blockIdx.x % kCl;
  r.hist = reinterpret_cast<unsigned*>(smem);
  r.list = reinterpret_cast<u64*>(smem);
  r.prefix = reinterpret_cast<double*>(smem) + kList;
  r.x = reinterpret_cast<float*>(smem + 2 * kBuckets * 4);
  r.lo = min(a.vocab, r.rank * slice);
  r.n = min(slice, a.vocab - r.lo);

  // the logits, and the best of them
  const T* from = static_cast<const T*>(a.logits) + (long long)row * a.stride + r.lo;
  float top = -INFINITY;
  int top_at = 0;
  auto take = [&](int i, float v) {
    v = v == v ? v + 0.0f : -INFINITY;  // -0 becomes +0: they tie
    r.x[i] = v;
    if (v > top) {
      top = v;
      top_at = i;
    }
  };
  constexpr int kVec = 16 / (int)sizeof(T);
  int i = 0;
  if (reinterpret_cast<uintptr_t>(from) % 16 == 0) {
    const int whole = r.n / kVec;
#pragma unroll 4
    for (int v = threadIdx.x; v < whole; v += kThreads) {
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(from) + v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) take(v * kVec + e, to_float(reinterpret_cast<const T*>(&b)[e]));
    }
    i = whole * kVec;
  }
#pragma unroll 8
  for (i += threadIdx.x; i < r.n; i += kThreads) take(i, to_float(from[i]));
  u64 best = top > -INFINITY ? order_of(top, r.lo + top_at) : 0;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, s));
  if (lane == 0) sh.warp_best[warp] = best;
  r.clear_histogram();  // ends with a barrier
  if (threadIdx.x < kCl) {
    for (int w = 0; w < kWarps; ++w) best = max(best, sh.warp_best[w]);
    r.at_rank(sh.best, threadIdx.x)[r.rank] = best;
  }
  r.sync_all();
  best = 0;
#pragma unroll
  for (int c = 0; c < kCl; ++c) best = max(best, sh.best[c]);

  const float t = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  if (best == 0 || !(t >= 1.17549435e-38f)) {
    if (r.rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = best == 0 ? -1 : index_of(best);
      if (a.probs) a.probs[row] = best == 0 ? 0.0f : 1.0f;
    }
    return;
  }
  r.scale = Scale(value_of(best), t);
  r.temperature = t;
  const float mp = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  r.least = mp;
  r.add_up({kHistogram, 0, kBuckets - 1, 0, 0});
  r.sync_all();
  if (r.rank == 0) {
    u64 order = best;
    double total = 1.0;
    r.lead(__ldg(a.uniforms + row), a.top_k ? __ldg(a.top_k + row) : 0, a.top_p ? __ldg(a.top_p + row) : 1.0f, mp, best, order,
           total);
    if (threadIdx.x == 0) {
      a.tokens[row] = index_of(order);
      if (a.probs) a.probs[row] = (float)(r.scale.weight(value_of(order)) / total);
    }
    if (kCl > 1) r.ask({kDone, 0, 0, 0, 0});
  } else {
    for (;;) {
      r.sync_all();
      const Command cmd = sh.command;
      if (cmd.op == kDone) break;
      r.serve(cmd);
      r.sync_all();
    }
  }
}

template <int kType, int kCl>
cudaError_t launch(const Sample& a, cudaStream_t s) {
  const int slice = ((a.vocab + kCl - 1) / kCl + 15) / 16 * 16;
  const int smem = 2 * kBuckets * 4 + slice * 4;
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<kType, kCl>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * kCl);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kCl;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = kCl > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel<kType, kCl>, a, slice);
}

template <int kType>
cudaError_t launch(const Sample& a, cudaStream_t s) {
  return a.vocab <= kOneCta ? launch<kType, 1>(a, s) : launch<kType, kCluster>(a, s);
}

}  // namespace

cudaError_t launch_sample(const Sample& a, int type, cudaStream_t s) {
  return type == 0 ? launch<0>(a, s) : type == 1 ? launch<1>(a, s) : launch<2>(a, s);
}

}  // namespace sampling
}  // namespace qb
