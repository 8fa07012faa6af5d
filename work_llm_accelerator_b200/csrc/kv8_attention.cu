// Decode attention over the 8-bit KV cache (include/qwen_b200_ops.h): one query row per new token, the row's
// own length, softmax in one pass with the running maximum and sum in fp32.
//
// Mathematics. With k_j = s_k c_j and v_j = s_v d_j (int8 codes, one scale per 64-token block) a score is
// (scale s_k) (q . c_j), and a tile of 32 tokens adds s_v sum_j p_j d_j: both products run on the codes, on
// mma.sync m16n8k16 in fp16, where a code is exact, and the scales multiply fp32 sums. q and the weights p would
// lose 13 bits in fp16, so each is the sum of two fp16 numbers, high + low (22 bits). A kv head serves at most 8
// query heads at a time, and the instruction has 16 rows: rows 0-7 hold the high parts, rows 8-15 the low ones, so
// the exact form costs no instruction more, and both halves of a sum meet in one thread. q is first scaled by a
// power of two per row (any fp32 size fits fp16); p is relative to its own tile's maximum, so that small weights of
// other tiles keep their bits, and the tile is joined to the running sums in fp32.
//
// Bound: HBM bytes of the cache (256 + 8/64 per token and kv head). Per tile and warp the arithmetic is 64 mma, ~350
// instructions of code conversion and ~100 of softmax, about a third of the issue slots at the memory's rate.
//
// Split: all (row, kv head) items lie end to end as tiles, in equal runs over the CTAs and in each CTA over its warps,
// whatever the lengths are. A warp streams its run through a ring of its own (cp.async, no CTA barrier in the loop).
// Items that a run cuts are joined in the CTA through shared memory, items that a CTA's run cuts by a second
// kernel, in the order of the tiles: results do not depend on timing.
#include <cuda_runtime.h>

#include "kv8_device.cuh"

namespace qb {
namespace kv8 {
namespace {

constexpr int kCtas = 148;  // one per SM; any number gives the same sums up to their split
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;    // tokens
constexpr int kStages = 3;   // 8 KB each: 128 KB in flight per SM, three times what the latency asks for
constexpr int kRows = 8;     // query heads of an item
constexpr int kTileBytes = kTile * kHead;       // of K or V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kPartFloats = kRows * (kHead + 2);  // sums [8][128], maxima [8], weights' sums [8]
constexpr int kMergeThreads = 256;

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

// Workspace: parts [2 * kCtas], then which item each part belongs to. Part 2 c: an item that began before CTA c's
// run (info = 2 * item + 1 if it ends there, else 2 * item; item = row * subs + sub); part 2 c + 1: one that began in it and goes on. -1: none.
constexpr size_t kInfoOffset = (size_t)2 * kCtas * kPartFloats * 4;
constexpr size_t kWorkBytes = kInfoOffset + 2 * kCtas * sizeof(int);

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum.
__device__ __forceinline__ void mma_first(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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

// Two codes to two fp16 numbers: with the sign bit flipped a code is c + 128, as the low byte of 0x64xx it is the
// number 1024 + 128 + c, and the subtraction is exact. `sel` places bytes 0, 1 (0x5150) or 2, 3 (0x5352).
template <unsigned kSel>
__device__ __forceinline__ unsigned codes_to_half2(unsigned flipped) {
  const unsigned n = __byte_perm(flipped, 0x64646464u, kSel);
  const unsigned bias = 0x64806480u;
  const __half2 r = __hsub2(reinterpret_cast<const __half2&>(n), reinterpret_cast<const __half2&>(bias));
  return reinterpret_cast<const unsigned&>(r);
}

// x, y -> their fp16 roundings and the fp16 roundings of what those leave
__device__ __forceinline__ void split_half(float x, float y, unsigned& high, unsigned& low) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  high = reinterpret_cast<const unsigned&>(h);
  low = reinterpret_cast<const unsigned&>(l);
}

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
  __device__ Layout(const Cache& c, const Attend& a)
      : group(a.q_heads / c.heads), chunks((group + kRows - 1) / kRows), subs(c.heads * chunks) {}
  __device__ int head(int sub) const { return sub / chunks; }
  __device__ int first_q(int sub) const { return head(sub) * group + sub % chunks * kRows; }
  __device__ int count(int sub) const { return min(kRows, group - sub % chunks * kRows); }
};

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

// This lane's dims of one query head, scaled by a power of two and split.
struct Query {
  unsigned f[8][4];  // dims 32 q4 + 4 s + {0, 1 | 2, 3} of head g, high and low
  float scale;       // scale * log2(e) * the power of two that was taken out
};

template <int kType>
__global__ void __launch_bounds__(kThreads, 1) split_kernel(Cache c, Attend a) {
  using T = typename TypeOf<kType>::T;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_sum[kWarps];
  __shared__ int4 start[kWarps];  // row, first tile among the row's, length, sequence
  __shared__ int part_item[2 * kWarps], part_ended[kWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q4 = lane % 4;
  const Layout lay(c, a);

  // ---- the runs: tiles before each thread's rows, the whole, and where this CTA's warps begin
  const int per_thread = (a.rows + kThreads - 1) / kThreads;
  const int row0 = min(a.rows, (int)threadIdx.x * per_thread), row1 = min(a.rows, row0 + per_thread);
  long long mine = 0;
  for (int r = row0; r < row1; ++r) mine += row_tiles(c, a, r);
  mine *= lay.subs;
  long long upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, i);
    if (lane >= i) upto += v;
  }
  if (lane == 31) warp_sum[warp] = upto;
  if (threadIdx.x < 2 * kWarps) part_item[threadIdx.x] = -1;
  __syncthreads();
  long long before = upto - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  const long long per_cta = max((long long)kWarps, (all + kCtas - 1) / kCtas);
  const long long cta0 = blockIdx.x * per_cta;
  const int cta_n = (int)max(0ll, min(per_cta, all - cta0));  // the entry point bounds all by 2^40
  const int per_warp = (cta_n + kWarps - 1) / kWarps;
  if (mine > 0 && before < cta0 + cta_n && before + mine > cta0) {
    long long pos = before;
    for (int r = row0; r < row1; ++r) {
      const long long n = (long long)row_tiles(c, a, r) * lay.subs;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const long long at = cta0 + w * per_warp;
        if (at >= pos && at < pos + n) start[w] = make_int4(r, (int)(at - pos), __ldg(a.row_len + r), __ldg(a.row_seq + r));
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
    auto load_query = [&](int it_row, int it_sub) {
      float4 x[8];
      float top = 0.0f;
      const T* from = static_cast<const T*>(a.q) + it_row * a.q_stride + (long long)(lay.first_q(it_sub) + g) * kHead + q4 * 32;
      const bool live = g < lay.count(it_sub);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        x[s] = live ? load4(from + s * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[s].x), fabsf(x[s].y)), fmaxf(fabsf(x[s].z), fabsf(x[s].w))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e and 2^e with the row's largest value in [1, 2) after the scaling
      const int e = top == 0.0f ? 127 : min(253, max(1, (int)(__float_as_uint(top) >> 23)));
      const float down = __uint_as_float((unsigned)(254 - e) << 23), up = __uint_as_float((unsigned)e << 23);
      q.scale = a.scale * up * 1.4426950408889634f;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        split_half(x[s].x * down, x[s].y * down, q.f[s][0], q.f[s][1]);
        split_half(x[s].z * down, x[s].w * down, q.f[s][2], q.f[s][3]);
      }
    };

    int it_row = row, it_sub = sub;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load(s);
    load_query(it_row, it_sub);  // while the first tiles are on their way

    float m = -INFINITY, l = 0.0f;  // head g: maximum (base 2) and this lane's share of the sum
    unsigned long long o[16];       // head g: dims 32 q4 + j and 32 q4 + 16 + j
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j] = 0;
    bool fresh = true, whole = false;
    int stage = 0;
    for (int t = 0; t < todo; ++t) {
      copies_wait<kStages - 2>();
      __syncwarp();
      const Note note = notes[stage];
      if (fresh) {
        fresh = false;
        whole = note.flags & kFirst;
        if (note.row != it_row || note.sub != it_sub) load_query(it_row = note.row, it_sub = note.sub);
      }
      const uint8_t* kt = ring + stage * kStageBytes;
      const uint8_t* vt = kt + kTileBytes;
      const float ks = note.flags & kBad ? __int_as_float(0x7fc00000) : scales[stage * 2], vs = scales[stage * 2 + 1];

      // scores of tokens 8 j + 2 q4 + {0, 1}: the contraction may take the dims in any order, so a lane's 32
      // codes of token 8 j + g are two 16-byte chunks, four codes for each of the 8 steps
      float s[4][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          b[j] = *reinterpret_cast<const uint4*>(kt + (j * 8 + g) * kHead + (((q4 * 2 + h) ^ g) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned w = reinterpret_cast<const unsigned*>(&b[j])[i] ^ 0x80808080u;
            const unsigned b0 = codes_to_half2<0x5150>(w), b1 = codes_to_half2<0x5352>(w);
            if (h == 0 && i == 0) mma_first(s[j], q.f[0], b0, b1);
            else mma(s[j], q.f[h * 4 + i], b0, b1);
          }
      }
      const float cs = q.scale * ks;
      float p[4][2], tm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) p[j][i] = (s[j][i] + s[j][i + 2]) * cs;
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

      // weights of two 8-token columns are the operand of one 16-token step
      unsigned pf[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        split_half(p[2 * k][0], p[2 * k][1], pf[k][0], pf[k][1]);
        split_half(p[2 * k + 1][0], p[2 * k + 1][1], pf[k][2], pf[k][3]);
      }
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
        float d[4][4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          unsigned b[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned x = reinterpret_cast<const unsigned*>(&raw[k][2 * i])[w];
            const unsigned y = reinterpret_cast<const unsigned*>(&raw[k][2 * i + 1])[w];
            const unsigned lo = __byte_perm(x, y, 0x5140) ^ 0x80808080u, hi = __byte_perm(x, y, 0x7362) ^ 0x80808080u;
            b[i][0] = codes_to_half2<0x5150>(lo);
            b[i][1] = codes_to_half2<0x5352>(lo);
            b[i][2] = codes_to_half2<0x5150>(hi);
            b[i][3] = codes_to_half2<0x5352>(hi);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (k == 0) mma_first(d[i], pf[0], b[0][i], b[1][i]);
            else mma(d[i], pf[1], b[0][i], b[1][i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[w * 4 + i] = fma2(av2, add2(pair(d[i][0], d[i][1]), pair(d[i][2], d[i][3])), mul2(o[w * 4 + i], keep2));
      }

      __syncwarp();  // the stage that is refilled next was read one step ago
      load(stage == 0 ? kStages - 1 : stage - 1);
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
          // an item that goes on: only at the end of the run, when the ring is free to take it
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
  int* info = reinterpret_cast<int*>(static_cast<uint8_t*>(a.work) + kInfoOffset) + 2 * blockIdx.x;
  const int my_item = lane < 2 * kWarps ? part_item[lane] : -1;
  const float* my_part = lane % 2 ? reinterpret_cast<const float*>(smem + lane / 2 % kWarps * kStages * kStageBytes)
                                  : reinterpret_cast<const float*>(smem + kPartsOffset) + lane / 2 % kWarps * kPartFloats;
  const unsigned live = __ballot_sync(0xffffffffu, my_item >= 0);
  const unsigned earlier = live & ((1u << lane) - 1);
  const int prev_item = __shfl_sync(0xffffffffu, my_item, earlier ? 31 - __clz(earlier) : 0);
  unsigned firsts = __ballot_sync(0xffffffffu, my_item >= 0 && !(earlier && prev_item == my_item));
  int before_info = -1, after_info = -1;
  while (firsts) {
    const int first = __ffs(firsts) - 1;
    firsts &= firsts - 1;
    const unsigned members = live & (firsts ? (firsts & -firsts) - 1 : ~0u) & ~((1u << first) - 1);
    const int last = 31 - __clz(members), item = __shfl_sync(0xffffffffu, my_item, first);
    const bool ended = last % 2 == 0 && part_ended[last / 2], done = first % 2 == 1 && ended;
    if (!done) {
      if (first % 2) after_info = item;
      else before_info = 2 * item + ended;
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
    for (unsigned rest = members; rest; rest &= rest - 1) {
      const int p = __ffs(rest) - 1;
      const float* x = p % 2 ? reinterpret_cast<const float*>(smem + p / 2 * kStages * kStageBytes)
                             : reinterpret_cast<const float*>(smem + kPartsOffset) + p / 2 * kPartFloats;
      const float4 v = *reinterpret_cast<const float4*>(x + warp * kHead + lane * 4);
      const float fp = __shfl_sync(0xffffffffu, f, p);
      o = make_float4(fmaf(fp, v.x, o.x), fmaf(fp, v.y, o.y), fmaf(fp, v.z, o.z), fmaf(fp, v.w, o.w));
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
  if (threadIdx.x == 0) {
    info[0] = before_info;
    info[1] = after_info;
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

// Joins the parts of an item that several CTAs' runs share: block (c, h) takes the item that began in CTA c and went
// on, head h of it. A warp takes every eighth part, its loads independent of one another.
template <int kType>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(Cache c, Attend a) {
  using T = typename TypeOf<kType>::T;
  constexpr int kMergeWarps = kMergeThreads / 32;
  __shared__ float4 sum[kMergeWarps][32];
  __shared__ float top[kMergeWarps], total[kMergeWarps], factor[kCtas];
  static_assert(kCtas <= kMergeThreads, "a thread per part");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float* work = static_cast<const float*>(a.work);
  const int* info = reinterpret_cast<const int*>(static_cast<const uint8_t*>(a.work) + kInfoOffset);
  const int cta = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int item = info[2 * cta + 1];
  if (item < 0) return;
  const Layout lay(c, a);
  const int it_row = item / lay.subs, it_sub = item - it_row * lay.subs;
  if (h >= lay.count(it_sub)) return;
  // part 0 is 2 cta + 1, part i the first one of CTA cta + i, up to the CTA where the item ends
  const int i = threadIdx.x, x = i > 0 && cta + i < kCtas ? info[2 * (cta + i)] : -1;
  const bool mine = i == 0 || x >> 1 == item;
  const float* my_part = work + (size_t)(i == 0 ? 2 * cta + 1 : 2 * (cta + i)) * kPartFloats;
  const float pm = mine ? my_part[kRows * kHead + h] : -INFINITY, pl = mine ? my_part[kRows * kHead + kRows + h] : 0.0f;
  float m = pm;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  if (lane == 0) top[warp] = m;
  const int n = __syncthreads_count(mine);
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) m = fmaxf(m, top[w]);
  const float f = mine ? ex2(pm - m) : 0.0f;
  if (i < kCtas) factor[i] = f;
  float l = mine ? f * pl : 0.0f;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
  if (lane == 0) total[warp] = l;
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 10
  for (int p = warp; p < n; p += kMergeWarps) {
    const float4 v = *reinterpret_cast<const float4*>(work + (size_t)(2 * (cta + p) + (p == 0)) * kPartFloats + h * kHead + lane * 4);
    const float fp = factor[p];
    o = make_float4(fmaf(fp, v.x, o.x), fmaf(fp, v.y, o.y), fmaf(fp, v.z, o.z), fmaf(fp, v.w, o.w));
  }
  sum[warp][lane] = o;
  __syncthreads();
  if (warp != 0) return;
  l = total[0];
#pragma unroll
  for (int w = 1; w < kMergeWarps; ++w) {
    const float4 v = sum[w][lane];
    l += total[w];
    o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
  }
  put_out<T>(a, it_row, lay.first_q(it_sub) + h, lane * 4, o, 1.0f / l);
  if (lane == 0) put_lse(a, it_row, lay.first_q(it_sub) + h, m, l);
}

template <int kType>
cudaError_t launch(const Cache& c, const Attend& a, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(split_kernel<kType>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return e;
  split_kernel<kType><<<kCtas, kThreads, kSmemBytes, s>>>(c, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCtas, kRows);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, merge_kernel<kType>, c, a);
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
