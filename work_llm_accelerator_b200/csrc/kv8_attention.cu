// Decode attention over the 8-bit KV cache (include/qwen_b200_ops.h): one query row per new token, the row's
// own length, softmax in one pass with the running maximum and sum in fp32.
//
// Mathematics. With k_j = s_k c_j and v_j = s_v d_j (int8 codes, one scale per 64-token block) a score is
// (scale s_k) (q . c_j), and a tile of 32 tokens adds s_v sum_j p_j d_j. Both sums run on the codes as they lie in the
// cache, on the int8 tensor cores (mma.sync m16n8k32): q, scaled by a power of two per row, and the weights p, relative
// to their own tile's maximum, are 31-bit integers X = x0 + 2^8 x1 + 2^16 x2 + 2^24 x3 with balanced int8 digits, so
// every digit product is exact in int32 and the rounding of X is at most 2^-30 of the row's largest |q|, or of the
// tile's largest weight: below the 2^-24 of fp32 itself for all that is not 64 times smaller. A kv head serves at most 8
// query heads at a time and the instruction has 16 rows: rows 0-7 hold digit 0 and rows 8-15 digit 1, whose products
// then meet in one thread; a second instruction holds digits 2 and 3 (three digits of 23 bits took as many instructions,
// 21.1 us where four take 21.5, and lost channels beside one that is 1000 times larger). An accumulator starts at the
// bits of 1.5 * 2^-6, whose last place is 2^-29: read as fp32 it is its integer in units of X, without a conversion.
// Each tile is joined to the running maximum and sums in fp32, so weights that are small beside another tile's keep
// their bits.
//
// Bound: HBM bytes of the cache (256 + 8/64 per token and kv head). Measured on B200 (12 heads on 2): 64 sequences x 2048
// 21.5 us (67.7 MB), of which the loop over the tiles takes 11, near the rate of HBM; the rest does not grow with the
// lengths: schedule 2.4, query and first tiles 2.7, join of the warps 1.9, launch. 1 x 131072 29.2 us (loop 15, join of
// the CTAs' parts 6), 1 x 517 10.7 us. On fp16 halves (m16n8k16) the codes' conversion cost 350 instructions per tile
// where three digits cost 64, and 64 x 2048 took 27.5 us (1 x 131072 26.8); tensor-map loads instead of cp.async took
// 0.5 us more.
//
// Split: all (row, kv head) items lie end to end as tiles, in equal runs over the CTAs and in each CTA over its warps,
// whatever the lengths are; a border that would cut an item moves to its beginning where that makes no run much longer.
// A warp streams its run through a ring of its own (cp.async, no CTA barrier in the loop).
// Items that a run cuts are joined in the CTA through shared memory; items that a CTA's run cuts by the CTA that
// finishes last, which flags in the workspace tell. Parts are joined in the order of the tiles: results do not
// depend on timing.
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>

#include "kv8_device.cuh"

namespace qb {
namespace kv8 {
namespace {

constexpr int kCtas = 148;  // one per SM; any number gives the same sums up to their split
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;    // tokens
constexpr int kStages = 3;   // 8 KB each: two tiles of every warp under way, 128 KB per SM
constexpr int kRows = 8;     // query heads of an item
constexpr int kMinRun = 16;  // tiles of a CTA's run, at least: two for each warp
constexpr int kSlack = 24;   // tiles by which a run may be longer to keep an item whole (about what a join costs)
constexpr int kTileBytes = kTile * kHead;       // of K or V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kPartFloats = kRows * (kHead + 2);  // sums [8][128], maxima [8], weights' sums [8]

// Shared memory: the rings, then a part per warp (an item that began before the warp's run), then the stage notes.
struct __align__(16) Note {
  int row, sub;  // the item
  int valid;     // tokens of the tile that the row reaches
  int flags;     // kFirst, kLast: the item's first and last tile; kBad: no such block
};
constexpr int kFirst = 1, kLast = 2, kBad = 4;
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kPartsOffset = kRingBytes;
constexpr int kNotesOffset = kPartsOffset + kWarps * kPartFloats * 4;
constexpr int kScalesOffset = kNotesOffset + kWarps * kStages * (int)sizeof(Note);
constexpr int kSmemBytes = kScalesOffset + kWarps * kStages * 2 * 4;
static_assert(kSmemBytes + 1024 <= 227 * 1024, "shared memory of one CTA, static part included");

// Workspace: parts [2 * kCtas], then a flag for each. Part 2 c: an item that began before CTA c's run; part 2 c + 1: one
// that began in it and goes on. The workspace may hold anything when a call begins, so a flag that is set holds the
// call's own 64-bit number. A CTA sets its part's flag and then looks at those of all the item's parts; at least the
// last one finds all of them set. Should two find that, both join the same parts in the same order and write the
// same bytes. Who joins takes the flags back: a graph's replays use one number, and find no flag set at their start.
typedef unsigned long long u64;
constexpr size_t kFlagsOffset = (size_t)2 * kCtas * kPartFloats * 4;
constexpr size_t kWorkBytes = kFlagsOffset + 2 * kCtas * sizeof(u64);

// One warp: sets flag `mine` of an item's n flags (its first at 0, the others at 1, 3, ...) and tells whether all are set.
__device__ __forceinline__ bool all_parts(u64* flags, u64 call, int mine, int n) {
  const int lane = threadIdx.x % 32;
  if (lane == 0) {
    __threadfence();  // the part itself first
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(flags + (mine ? 2 * mine - 1 : 0)), "l"(call) : "memory");
  }
  __syncwarp();
  __threadfence();  // sequentially consistent: of two CTAs that set and look, one sees the other's
  bool all = true;
  for (int i = lane; i < n; i += 32) {
    u64 x;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(x) : "l"(flags + (i ? 2 * i - 1 : 0)) : "memory");
    all = all && x == call;
  }
  all = __all_sync(0xffffffffu, all);
  if (all) {
    for (int i = lane; i < n; i += 32)
      asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(flags + (i ? 2 * i - 1 : 0)), "l"(0ull) : "memory");
    __threadfence();  // the parts are read behind the flags
  }
  return all;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// d = a b + d on int8 codes; mma_first: d = a b + the bits of kZero.
__device__ __forceinline__ void mma(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr float kUnits = 536870912.0f;  // 2^29: X of 1
constexpr float kZero = 1.5f / 64.0f;   // kZero + n / kUnits for |n| < 2^22 has the bits of kZero plus n
constexpr int kZeroBits = 0x3cc00000;
__device__ __forceinline__ void mma_first(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                          unsigned b1, const int (&zero)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(zero[0]), "r"(zero[1]), "r"(zero[2]), "r"(zero[3]));
}

// Pairs of fp32 numbers in one instruction.
__device__ __forceinline__ unsigned long long pair(float x, float y) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Digits of x in [-2, 2]: the bytes of X + 0x808080 are the lower digits + 128 and the top one, and flipping the top bits of
// the lower ones makes them int8.
__device__ __forceinline__ unsigned digits(float x) {
  return ((unsigned)__float2int_rn(x * kUnits) + 0x00808080u) ^ 0x00808080u;
}
// 4 x 4 bytes transposed: byte i of the four words to word i. Of numbers to digits, of tokens to dims.
__device__ __forceinline__ void transpose(unsigned x0, unsigned x1, unsigned x2, unsigned x3, unsigned (&d)[4]) {
  const unsigned l0 = __byte_perm(x0, x1, 0x5140), h0 = __byte_perm(x0, x1, 0x7362);
  const unsigned l1 = __byte_perm(x2, x3, 0x5140), h1 = __byte_perm(x2, x3, 0x7362);
  d[0] = __byte_perm(l0, l1, 0x5410);
  d[1] = __byte_perm(l0, l1, 0x7632);
  d[2] = __byte_perm(h0, h1, 0x5410);
  d[3] = __byte_perm(h0, h1, 0x7632);
}
// Two columns' digit sums to two fp32 numbers: lo is (digit 0, digit 1) of both, hi (digit 2, digit 3), each kZero off. The
// 256 folds the lower digit's kZero into the upper one's difference, which stays exact; three roundings of 2^-24 follow.
__device__ __forceinline__ u64 join_digits(const int (&lo)[4], const int (&hi)[4]) {
  constexpr float kBoth = -(kZero + kZero / 256.0f);
  auto join = [](const int(&d)[4]) {
    return fma2(add2(pair(__int_as_float(d[2]), __int_as_float(d[3])), pair(kBoth, kBoth)), pair(256.0f, 256.0f),
                pair(__int_as_float(d[0]), __int_as_float(d[1])));
  };
  return fma2(join(hi), pair(65536.0f, 65536.0f), join(lo));
}

__device__ __forceinline__ unsigned word(const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

__device__ __forceinline__ void copy16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Items of a row: kv heads x chunks of at most 8 query heads.
struct Layout {
  int group, chunks, subs;
  Layout(const Cache& c, const Attend& a)
      : group(a.q_heads / c.heads), chunks((group + kRows - 1) / kRows), subs(c.heads * chunks) {}
  __device__ int head(int sub) const { return sub / chunks; }
  __device__ int first_q(int sub) const { return head(sub) * group + sub % chunks * kRows; }
  __device__ int count(int sub) const { return min(kRows, group - sub % chunks * kRows); }
};

// x / size for a quotient below 2^20, without the long division.
__device__ __forceinline__ int run_of(long long x, long long size) {
  int c = (int)((float)x / (float)size);
  while (c * size > x) --c;
  while ((c + 1) * size <= x) ++c;
  return c;
}

enum RowKind { kSkip, kEmpty, kWrong, kLive };
__device__ __forceinline__ RowKind row_kind(const Cache& c, int seq, int len) {
  if (seq < 0) return kSkip;
  if (seq >= c.n_seqs || len < 0 || len > (long long)c.width * kBlock) return kWrong;
  return len == 0 ? kEmpty : kLive;
}
__device__ __forceinline__ int row_tiles(const Cache& c, const Attend& a, int row) {
  const int len = __ldg(a.row_len + row);
  return row_kind(c, __ldg(a.row_seq + row), len) == kLive ? (len - 1) / kTile + 1 : 0;
}

// Four results of one head: the sums over the weights' sum, rounded once.
template <typename T>
__device__ __forceinline__ void put_out(const Attend& a, long long row, int h, int dim, float4 o, float r) {
  store4(static_cast<T*>(a.out) + row * a.out_stride + (long long)h * kHead + dim,
         make_float4(o.x * r, o.y * r, o.z * r, o.w * r));
}
__device__ __forceinline__ void put_lse(const Attend& a, long long row, int h, float m, float l) {
  if (a.lse) a.lse[row * a.q_heads + h] = m * 0.6931471805599453f + logf(l);
}

// This lane's dims of one query head as digits, and what a score of them is multiplied by.
struct Query {
  unsigned d[8][4];  // dims 32 q4 + 4 i + {0 .. 3} of head g
  float scale;       // scale * log2(e) * the power of two that was taken out
};

template <int kType>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(Cache c, Attend a, Layout lay, u64 call) {
  using T = typename TypeOf<kType>::T;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_sum[kWarps], part_from[kWarps], border[2];
  __shared__ unsigned warp_least[kWarps], warp_most[kWarps];
  __shared__ int4 start[kWarps];  // row, first tile among the row's, length, sequence
  __shared__ int part_item[2 * kWarps], part_ended[kWarps];
  __shared__ int2 join[2];  // an item whose parts are joined here: its first CTA, and how many have a part
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q4 = lane % 4;

  // ---- the runs: tiles before each thread's rows, the whole, and where this CTA's warps begin
  const int per_thread = (a.rows + kThreads - 1) / kThreads;
  const int row0 = min(a.rows, (int)threadIdx.x * per_thread), row1 = min(a.rows, row0 + per_thread);
  long long mine = 0;
  unsigned least = ~0u, most = 0;
  for (int r = row0; r < row1; ++r) {
    const unsigned n = row_tiles(c, a, r);
    mine += n;
    least = min(least, n - 1);  // rows without a tile are not among them
    most = max(most, n);
  }
  mine *= lay.subs;
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  long long upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, i);
    if (lane >= i) upto += v;
  }
  if (lane == 31) {
    warp_sum[warp] = upto;
    warp_least[warp] = least;
    warp_most[warp] = most;
  }
  if (threadIdx.x < 2 * kWarps) part_item[threadIdx.x] = -1;
  __syncthreads();
  long long before = upto - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
    least = min(least, warp_least[w]);
    most = max(most, warp_most[w]);
  }
  ++least;
  // Run c begins at tile c * per_cta, or at the beginning of the item there if that stays whole: it is short, or all
  // are as long and a little longer than a run, so that a run gets one of them or none.
  const long long per_cta = max((long long)kMinRun, (all + kCtas - 1) / kCtas);
  const bool alike = least == most && most >= per_cta && most <= per_cta + kSlack;
  if (threadIdx.x < 2) border[threadIdx.x] = all;
  __syncthreads();
  if (mine > 0) {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const long long at = (blockIdx.x + i) * per_cta;
      if (at < before || at >= before + mine) continue;
      long long pos = before;
      for (int r = row0; r < row1; ++r) {
        const int tiles = row_tiles(c, a, r);
        const long long n = (long long)tiles * lay.subs;
        if (at < pos + n) {
          border[i] = tiles <= kSlack || alike ? at - (int)(at - pos) % tiles : at;
          break;
        }
        pos += n;
      }
    }
  }
  __syncthreads();
  const long long cta0 = border[0];
  const int cta_n = (int)(border[1] - cta0);  // the entry point bounds all by 2^37
  const int per_warp = (cta_n + kWarps - 1) / kWarps;
  if (mine > 0 && before < cta0 + cta_n && before + mine > cta0) {
    long long pos = before;
    for (int r = row0; r < row1; ++r) {
      const long long n = (long long)row_tiles(c, a, r) * lay.subs;
      if (pos + n > cta0 && pos < cta0 + cta_n) {
        const int4 row = make_int4(r, 0, __ldg(a.row_len + r), __ldg(a.row_seq + r));
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const long long at = cta0 + w * per_warp;
          if (at >= pos && at < pos + n) start[w] = make_int4(row.x, (int)(at - pos), row.z, row.w);
        }
      }
      pos += n;
    }
  }
  __syncthreads();

  // ---- this warp's run
  const int todo = max(0, min(per_warp, cta_n - warp * per_warp));
  uint8_t* ring = smem + warp * kStages * kStageBytes;
  float* part = reinterpret_cast<float*>(smem + kPartsOffset) + warp * kPartFloats;
  Note* notes = reinterpret_cast<Note*>(smem + kNotesOffset) + warp * kStages;
  float* scales = reinterpret_cast<float*>(smem + kScalesOffset) + warp * kStages * 2;
  if (todo > 0) {
    // the load cursor
    int row = start[warp].x, len = start[warp].z, tiles = (len - 1) / kTile + 1;
    int sub = start[warp].y / tiles, tile = start[warp].y - sub * tiles, left = todo;
    int head = sub / lay.chunks, chunk = sub - head * lay.chunks;
    const int* table = c.table + (long long)start[warp].w * c.width;
    int block = __ldg(table + tile / (kBlock / kTile));

    // a copy: 4 tokens x 8 chunks of 16 bytes; chunk x of token t lies at x ^ (t % 8), so that fragments are read
    // without bank conflicts
    const int lane_token = lane / 8;
    const unsigned to_even = smem_u32(ring) + lane_token * kHead + (((lane % 8) ^ lane_token) << 4);
    const unsigned to_odd = to_even ^ 64;
    auto load = [&](int stage) {
      if (left > 0) {
        const bool bad = (unsigned)block >= (unsigned)c.n_blocks;
        const long long at = (long long)(bad ? 0 : block) * c.heads + head;
        const int valid = min(kTile, len - tile * kTile);
        if (lane == 0) {
          notes[stage] = {row, sub, valid, (tile == 0 ? kFirst : 0) | (tile == tiles - 1 ? kLast : 0) | (bad ? kBad : 0)};
          if (bad) bad_index();
        }
        if (lane < 2) copy4(smem_u32(scales + stage * 2 + lane), (lane ? c.scales[1] : c.scales[0]) + at);
        const long long from = at * (kBlock * kHead) + tile % (kBlock / kTile) * kTileBytes + lane * 16;
        const int8_t* k = c.codes[0] + from;
        const int8_t* v = c.codes[1] + from;
        const unsigned off = stage * kStageBytes;
        if (valid == kTile) {
#pragma unroll
          for (int i = 0; i < kTile / 4; ++i) {
            const unsigned to = (i % 2 ? to_odd : to_even) + off + i * 4 * kHead;
            copy16(to, k + i * 4 * kHead);
            copy16(to + kTileBytes, v + i * 4 * kHead);
          }
        } else {
          for (int i = 0; i < kTile / 4; ++i) {
            const unsigned to = (i % 2 ? to_odd : to_even) + off + i * 4 * kHead;
            if (i * 4 + lane_token < valid) {
              copy16(to, k + i * 4 * kHead);
              copy16(to + kTileBytes, v + i * 4 * kHead);
            }
          }
        }
        // the next tile, its block's id one step ahead of its use
        if (--left > 0) {
          if (++tile == tiles) {
            tile = 0;
            ++sub;
            if (++chunk == lay.chunks) {
              chunk = 0;
              if (++head == c.heads) {
                head = sub = 0;
                do {
                  ++row;
                  tiles = row_tiles(c, a, row);
                } while (tiles == 0);
                len = __ldg(a.row_len + row);
                table = c.table + (long long)__ldg(a.row_seq + row) * c.width;
              }
            }
          }
          block = __ldg(table + tile / (kBlock / kTile));
        }
      }
      copies_commit();
    };

    Query q;
    auto load_query = [&](int it_row, int it_sub, auto meanwhile) {
      float4 x[8];
      unsigned top = 0;
      const T* from = static_cast<const T*>(a.q) + it_row * a.q_stride + (long long)(lay.first_q(it_sub) + g) * kHead + q4 * 32;
      const bool live = g < lay.count(it_sub);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = live ? load4(from + i * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      meanwhile();
#pragma unroll
      for (int i = 0; i < 8; ++i)
        top = max(top, max(max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu),
                           max(__float_as_uint(x[i].z) & 0x7fffffffu, __float_as_uint(x[i].w) & 0x7fffffffu)));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row's largest value is in [1, 2) after the scaling, in [0.5, 1) and doubled where 2^-127, which is no normal
      // number, would be asked for; a NaN or an infinity in the row makes all its scores NaN
      const int e = top == 0 ? 127 : min(254, max(1, (int)(top >> 23)));
      const float down = __uint_as_float((unsigned)max(1, 254 - e) << 23), up = __uint_as_float((unsigned)e << 23);
      const float half = e == 254 ? 0.5f : 1.0f;
      q.scale = top >= 0x7f800000u ? __int_as_float(0x7fc00000) : up * 1.4426950408889634f * a.scale;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        transpose(digits(x[i].x * down * half), digits(x[i].y * down * half), digits(x[i].z * down * half),
                  digits(x[i].w * down * half), q.d[i]);
    };

    int it_row = row, it_sub = sub;
    // the query's loads go first: behind the first tiles' they would wait for 19 MB to come in
    load_query(it_row, it_sub, [&] {
#pragma unroll 1
      for (int s = 0; s < kStages - 1; ++s) load(s);
    });

    float m = -INFINITY, l = 0.0f;  // head g: maximum (base 2) and this lane's share of the sum
    unsigned long long o[16];       // head g: dims 32 q4 + j and 32 q4 + 16 + j
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = 0;
    bool fresh = true, whole = false;
    int stage = 0, began = 0;
    const int zero[4] = {kZeroBits, kZeroBits, kZeroBits, kZeroBits};
    for (int t = 0; t < todo; ++t) {
      copies_wait<kStages - 2>();
      __syncwarp();  // all lanes' copies are here, and all lanes are done with the stage before, which is refilled
      load(stage == 0 ? kStages - 1 : stage - 1);
      const Note note = notes[stage];
      if (fresh) {
        fresh = false;
        began = t;
        whole = note.flags & kFirst;
        if (note.row != it_row || note.sub != it_sub) load_query(it_row = note.row, it_sub = note.sub, [] {});
      }
      const uint8_t* kt = ring + stage * kStageBytes;
      const uint8_t* vt = kt + kTileBytes;
      const float ks = note.flags & kBad ? __int_as_float(0x7fc00000) : scales[stage * 2], vs = scales[stage * 2 + 1];

      // scores of tokens 8 j + 2 q4 + {0, 1}: the contraction may take the dims in any order, so a lane's 32
      // codes of token 8 j + g are two 16-byte chunks, eight codes for each of the 4 steps
      int lo[4][4], hi[4][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          b[j] = *reinterpret_cast<const uint4*>(kt + (j * 8 + g) * kHead + (((q4 * 2 + h) ^ g) << 4));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned(&x)[4] = q.d[h * 4 + i * 2], (&y)[4] = q.d[h * 4 + i * 2 + 1];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned b0 = i ? b[j].z : b[j].x, b1 = i ? b[j].w : b[j].y;
            if (h == 0 && i == 0) {
              mma_first(lo[j], x[0], x[1], y[0], y[1], b0, b1, zero);
              mma_first(hi[j], x[2], x[3], y[2], y[3], b0, b1, zero);
            } else {
              mma(lo[j], x[0], x[1], y[0], y[1], b0, b1);
              mma(hi[j], x[2], x[3], y[2], y[3], b0, b1);
            }
          }
        }
      }
      const float cs = q.scale * ks;
      float p[4][2], tm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 s = unpair(mul2(join_digits(lo[j], hi[j]), pair(cs, cs)));
        p[j][0] = s.x;
        p[j][1] = s.y;
      }
      if (note.valid < kTile) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (j * 8 + q4 * 2 + i >= note.valid) p[j][i] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) tm = fmaxf(tm, fmaxf(p[j][0], p[j][1]));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
      float tl = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) p[j][i] = ex2(p[j][i] - tm);
        tl += p[j][0] + p[j][1];
      }
      const float mn = fmaxf(m, tm), keep = ex2(m - mn), add = ex2(tm - mn), av = add * vs;
      m = mn;
      l = l * keep + add * tl;
      const unsigned long long keep2 = pair(keep, keep), av2 = pair(av, av);

      // this lane's weights are what it holds of the operand
      unsigned pd[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        transpose(digits(p[2 * k][0]), digits(p[2 * k][1]), digits(p[2 * k + 1][0]), digits(p[2 * k + 1][1]), pd[k]);
      uint4 raw[2][4];  // dims 16 g .. 16 g + 15 of tokens 16 k + 2 q4 + {0, 1, 8, 9}
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int token = k * 16 + q4 * 2 + i % 2 + i / 2 * 8;
          raw[k][i] = *reinterpret_cast<const uint4*>(vt + token * kHead + ((g ^ (q4 * 2 + i % 2)) << 4));
        }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        unsigned b[2][4];  // from four dims of a token to four tokens of a dim
#pragma unroll
        for (int k = 0; k < 2; ++k)
          transpose(word(raw[k][0], w), word(raw[k][1], w), word(raw[k][2], w), word(raw[k][3], w), b[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          int dl[4], dh[4];
          mma_first(dl, pd[0][0], pd[0][1], pd[1][0], pd[1][1], b[0][i], b[1][i], zero);
          mma_first(dh, pd[0][2], pd[0][3], pd[1][2], pd[1][3], b[0][i], b[1][i], zero);
          o[w * 4 + i] = fma2(av2, join_digits(dl, dh), mul2(o[w * 4 + i], keep2));
        }
      }

      stage = stage + 1 == kStages ? 0 : stage + 1;

      const bool ends = note.flags & kLast;
      if (ends || t == todo - 1) {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (whole && ends) {
          if (g < lay.count(it_sub)) {
            const int h = lay.first_q(it_sub) + g;
            const float r = 1.0f / l;
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float2 x[4] = {unpair(o[j]), unpair(o[j + 1]), unpair(o[j + 2]), unpair(o[j + 3])};
              put_out<T>(a, it_row, h, q4 * 32 + j, make_float4(x[0].x, x[1].x, x[2].x, x[3].x), r);
              put_out<T>(a, it_row, h, q4 * 32 + 16 + j, make_float4(x[0].y, x[1].y, x[2].y, x[3].y), r);
            }
            if (q4 == 0) put_lse(a, it_row, h, m, l);
          }
        } else {
          // an item that goes on: only at the end of the run, when the ring is free to take it once all lanes have read
          if (whole) {
            copies_wait<0>();
            __syncwarp();
          }
          float* to = whole ? reinterpret_cast<float*>(ring) : part;
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float2 x[4] = {unpair(o[j]), unpair(o[j + 1]), unpair(o[j + 2]), unpair(o[j + 3])};
            *reinterpret_cast<float4*>(to + g * kHead + q4 * 32 + j) = make_float4(x[0].x, x[1].x, x[2].x, x[3].x);
            *reinterpret_cast<float4*>(to + g * kHead + q4 * 32 + 16 + j) = make_float4(x[0].y, x[1].y, x[2].y, x[3].y);
          }
          if (q4 == 0) {
            to[kRows * kHead + g] = m;
            to[kRows * kHead + kRows + g] = l;
          }
          if (lane == 0) {
            part_item[2 * warp + whole] = it_row * lay.subs + it_sub;
            if (!whole) part_ended[warp] = ends;
            else part_from[warp] = cta0 + warp * per_warp + began;
          }
        }
        fresh = true;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = 0;
      }
    }
    copies_wait<0>();
  }
  __syncthreads();

  // ---- join the warps' parts, warp h head h: part 2 w is warp w's item from before, part 2 w + 1 the one that goes on
  const int my_item = lane < 2 * kWarps ? part_item[lane] : -1;
  const float* my_part = lane % 2 ? reinterpret_cast<const float*>(smem + lane / 2 % kWarps * kStages * kStageBytes)
                                  : reinterpret_cast<const float*>(smem + kPartsOffset) + lane / 2 % kWarps * kPartFloats;
  const unsigned live = __ballot_sync(0xffffffffu, my_item >= 0);
  const unsigned earlier = live & ((1u << lane) - 1);
  const int prev_item = __shfl_sync(0xffffffffu, my_item, earlier ? 31 - __clz(earlier) : 0);
  unsigned firsts = __ballot_sync(0xffffffffu, my_item >= 0 && !(earlier && prev_item == my_item));
  int open_item[2] = {-1, -1}, after_warp = 0;  // from before and not done here; going on
  while (firsts) {
    const int first = __ffs(firsts) - 1;
    firsts &= firsts - 1;
    const unsigned members = live & (firsts ? (firsts & -firsts) - 1 : ~0u) & ~((1u << first) - 1);
    const int last = 31 - __clz(members), item = __shfl_sync(0xffffffffu, my_item, first);
    const bool ended = last % 2 == 0 && part_ended[last / 2], done = first % 2 == 1 && ended;
    if (!done) {
      open_item[first % 2] = item;
      if (first % 2) after_warp = first / 2;
    }
    const int it_row = item / lay.subs, it_sub = item - it_row * lay.subs;
    if (warp >= lay.count(it_sub)) continue;
    const bool member = members >> lane & 1;
    const float pm = member ? my_part[kRows * kHead + warp] : -INFINITY;
    float m = pm;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
    const float f = member ? ex2(pm - m) : 0.0f;
    float l = member ? f * my_part[kRows * kHead + kRows + warp] : 0.0f;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (unsigned rest = members; rest;) {
      float4 v[kWarps];
      float fp[kWarps];
#pragma unroll
      for (int i = 0; i < kWarps; ++i, rest &= rest - 1) {  // a part too many counts 0 times
        const int p = rest ? __ffs(rest) - 1 : first;
        const float* x = p % 2 ? reinterpret_cast<const float*>(smem + p / 2 * kStages * kStageBytes)
                               : reinterpret_cast<const float*>(smem + kPartsOffset) + p / 2 * kPartFloats;
        v[i] = *reinterpret_cast<const float4*>(x + warp * kHead + lane * 4);
        fp[i] = __shfl_sync(0xffffffffu, f, p);
        if (!rest) v[i] = make_float4(0.f, 0.f, 0.f, 0.f), fp[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kWarps; ++i)
        o = make_float4(fmaf(fp[i], v[i].x, o.x), fmaf(fp[i], v[i].y, o.y), fmaf(fp[i], v[i].z, o.z), fmaf(fp[i], v[i].w, o.w));
    }
    if (done) {
      put_out<T>(a, it_row, lay.first_q(it_sub) + warp, lane * 4, o, 1.0f / l);
      if (lane == 0) put_lse(a, it_row, lay.first_q(it_sub) + warp, m, l);
    } else {
      float* to = static_cast<float*>(a.work) + (size_t)(2 * blockIdx.x + first % 2) * kPartFloats;
      *reinterpret_cast<float4*>(to + warp * kHead + lane * 4) = o;
      if (lane == 0) {
        to[kRows * kHead + warp] = m;
        to[kRows * kHead + kRows + warp] = l;
      }
    }
  }

  // ---- join an item's parts over the CTAs, in the one that finishes last: a CTA has a part of at most two
  if (open_item[0] >= 0 || open_item[1] >= 0) {
    __syncthreads();
    if (warp < 2) {
      const int item = warp ? open_item[1] : open_item[0];
      bool last = false;
      if (item >= 0) {
        // the item's tiles begin at `from`: in which CTA, and in how many
        const int tiles = row_tiles(c, a, item / lay.subs);
        const long long from = warp ? part_from[after_warp] : cta0 - start[0].y % tiles;
        const int first_cta = run_of(from, per_cta), n = run_of(from + tiles - 1, per_cta) - first_cta + 1;
        // its flags: that of part 2 first_cta + 1, then of every second one
        u64* flags = reinterpret_cast<u64*>(static_cast<uint8_t*>(a.work) + kFlagsOffset) + 2 * first_cta + 1;
        last = all_parts(flags, call, (int)blockIdx.x - first_cta, n);
        if (lane == 0) join[warp] = make_int2(first_cta, n);
      }
      if (lane == 0 && !last) join[warp] = make_int2(0, 0);
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int item = which ? open_item[1] : open_item[0];
    if (item < 0) continue;
    const int it_row = item / lay.subs, it_sub = item - it_row * lay.subs, first_cta = join[which].x, n = join[which].y;
    if (n == 0 || warp >= lay.count(it_sub)) continue;
    __syncwarp();  // the factors of another item
    // a factor per part, in the ring's place; a batch of parts is loaded at once, the first beside the maxima
    const float* parts = static_cast<const float*>(a.work) + (size_t)2 * first_cta * kPartFloats;
    auto part = [&](int i) { return parts + (size_t)(2 * i + (i == 0)) * kPartFloats; };
    float* factor = reinterpret_cast<float*>(smem) + warp * kCtas;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAhead = 32;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += kAhead) {
      float4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < n) v[i] = __ldcg(reinterpret_cast<const float4*>(part(i0 + i) + warp * kHead + lane * 4));
      if (i0 == 0) {
        for (int i = lane; i < n; i += 32) {
          factor[i] = __ldcg(part(i) + kRows * kHead + warp);
          m = fmaxf(m, factor[i]);
        }
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
        for (int i = lane; i < n; i += 32) {
          factor[i] = ex2(factor[i] - m);
          l = fmaf(factor[i], __ldcg(part(i) + kRows * kHead + kRows + warp), l);
        }
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < n) {
          const float f = factor[i0 + i];
          o = make_float4(fmaf(f, v[i].x, o.x), fmaf(f, v[i].y, o.y), fmaf(f, v[i].z, o.z), fmaf(f, v[i].w, o.w));
        }
    }
    put_out<T>(a, it_row, lay.first_q(it_sub) + warp, lane * 4, o, 1.0f / l);
    if (lane == 0) put_lse(a, it_row, lay.first_q(it_sub) + warp, m, l);
  }

  // ---- rows without a tile: nothing cached yet, or an index that is no row of the cache
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const RowKind kind = row_kind(c, __ldg(a.row_seq + r), __ldg(a.row_len + r));
    if (kind == kLive || kind == kSkip) continue;
    const float x = kind == kEmpty ? 0.0f : __int_as_float(0x7fc00000);
    if (kind == kWrong && threadIdx.x == 0) bad_index();
    for (int i = threadIdx.x; i < a.q_heads * kHead / 4; i += kThreads)
      put_out<T>(a, r, 0, i * 4, make_float4(x, x, x, x), 1.0f);
    if (a.lse)
      for (int h = threadIdx.x; h < a.q_heads; h += kThreads)
        a.lse[(long long)r * a.q_heads + h] = kind == kEmpty ? -INFINITY : x;
  }
}

// A number for a call, in the upper 48 bits: a counter through the finaliser of splitmix64 (Steele, Lea and Flood, 2014).
u64 call_number() {
  static std::atomic<u64> next{(u64)std::chrono::steady_clock::now().time_since_epoch().count()};
  u64 x = next.fetch_add(0x9e3779b97f4a7c15ull);
  x = (x ^ (x >> 30)) * 0xbf58476d1ce4e5b9ull;
  x = (x ^ (x >> 27)) * 0x94d049bb133111ebull;
  x = (x ^ (x >> 31)) & ~0xffffull;
  return x ? x : 1ull << 16;
}

template <int kType>
cudaError_t launch(const Cache& c, const Attend& a, cudaStream_t s) {
  const cudaError_t e =
      cudaFuncSetAttribute(attention_kernel<kType>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return e;
  attention_kernel<kType><<<kCtas, kThreads, kSmemBytes, s>>>(c, a, Layout(c, a), call_number());
  return cudaGetLastError();
}

}  // namespace

size_t attention_workspace(int, int, int) { return kWorkBytes; }

cudaError_t launch_attention(const Cache& c, const Attend& a, int type, cudaStream_t s) {
  return type == 0 ? launch<0>(c, a, s) : type == 1 ? launch<1>(c, a, s) : launch<2>(c, a, s);
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
