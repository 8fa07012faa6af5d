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
constexpr int kMergeThreads = 128;

// Shared memory: the rings, then a part per warp (an item that began before the warp's run), then the stage notes.
struct Note {
  long long item;  // row * subs + sub
  int valid;       // tokens of the tile that the row reaches
  int flags;       // kFirst, kLast: the item's first and last tile; kBad: no such block
};
constexpr int kFirst = 1, kLast = 2, kBad = 4;
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kPartsOffset = kRingBytes;
constexpr int kNotesOffset = kPartsOffset + kWarps * kPartFloats * 4;
constexpr int kScalesOffset = kNotesOffset + kWarps * kStages * (int)sizeof(Note);
constexpr int kSmemBytes = kScalesOffset + kWarps * kStages * 2 * 4;
static_assert(kSmemBytes + 1024 <= 227 * 1024, "shared memory of one CTA, static part included");

// Workspace: parts [2 * kCtas], then which item each part belongs to. Part 2 c: an item that began before CTA c's
// run (info = 2 * item + 1 if it ends there, else 2 * item); part 2 c + 1: one that began in it and goes on. -1: none.
constexpr size_t kInfoOffset = (size_t)2 * kCtas * kPartFloats * 4;
constexpr size_t kWorkBytes = kInfoOffset + 2 * kCtas * sizeof(long long);

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

template <int kType>
__global__ void __launch_bounds__(kThreads, 1) split_kernel(Cache c, Attend a) {
  using T = typename TypeOf<kType>::T;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_sum[kWarps], start_off[kWarps], part_item[kWarps][2];
  __shared__ int start_row[kWarps], part_ended[kWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q4 = lane % 4;
  const Layout lay(c, a);
  float* work = static_cast<float*>(a.work);
  long long* info = reinterpret_cast<long long*>(static_cast<uint8_t*>(a.work) + kInfoOffset);

  // ---- the runs: tiles before each thread's rows, the whole, and where this CTA's warps begin
  const int per_thread = (a.rows + kThreads - 1) / kThreads;
  const int row0 = min(a.rows, (int)threadIdx.x * per_thread), row1 = min(a.rows, row0 + per_thread);
  long long mine = 0;
  for (int r = row0; r < row1; ++r) mine += row_tiles(c, a, r);
  long long upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, i);
    if (lane >= i) upto += v;
  }
  if (lane == 31) warp_sum[warp] = upto;
  if (threadIdx.x < 2 * kWarps) part_item[threadIdx.x / 2][threadIdx.x % 2] = -1;
  __syncthreads();
  long long before = upto - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  all *= lay.subs;
  const long long per_cta = max((long long)kWarps, (all + gridDim.x - 1) / gridDim.x);
  const long long cta0 = blockIdx.x * per_cta;
  const long long cta_n = max(0ll, min(per_cta, all - cta0));
  const long long per_warp = (cta_n + kWarps - 1) / kWarps;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const long long at = cta0 + w * per_warp;
    if (mine > 0 && at >= before * lay.subs && at < (before + mine) * lay.subs) {
      long long pos = before * lay.subs;
      int r = row0;
      for (; r < row1; ++r) {
        const long long n = (long long)row_tiles(c, a, r) * lay.subs;
        if (at < pos + n) break;
        pos += n;
      }
      start_row[w] = r;
      start_off[w] = at - pos;
    }
  }
  __syncthreads();

  // ---- this warp's run
  const long long todo = max(0ll, min(per_warp, cta_n - warp * per_warp));
  uint8_t* ring = smem + warp * kStages * kStageBytes;
  float* part = reinterpret_cast<float*>(smem + kPartsOffset) + warp * kPartFloats;
  Note* notes = reinterpret_cast<Note*>(smem + kNotesOffset) + warp * kStages;
  float* scales = reinterpret_cast<float*>(smem + kScalesOffset) + warp * kStages * 2;
  if (todo > 0) {
    // the load cursor
    int row = start_row[warp], len = __ldg(a.row_len + row), tiles = (len - 1) / kTile + 1;
    int sub = (int)(start_off[warp] / tiles), tile = (int)(start_off[warp] % tiles);
    const int* table = c.table + (long long)__ldg(a.row_seq + row) * c.width;
    long long left = todo;
    int block = __ldg(table + tile / (kBlock / kTile));

    const int lane_token = lane / 8, lane_chunk = lane % 8;  // a copy: 4 tokens x 8 chunks of 16 bytes
    auto load = [&](int stage) {
      if (left > 0) {
        const bool bad = block < 0 || block >= c.n_blocks;
        const long long at = (long long)(bad ? 0 : block) * c.heads + lay.head(sub);
        const int valid = min(kTile, len - tile * kTile);
        if (lane == 0) {
          notes[stage] = {(long long)row * lay.subs + sub, valid,
                          (tile == 0 ? kFirst : 0) | (tile == tiles - 1 ? kLast : 0) | (bad ? kBad : 0)};
          if (bad) bad_index();
        }
        if (lane < 2) copy4(smem_u32(scales + stage * 2 + lane), c.scales[lane] + at);
        const long long from = (at * kBlock + tile % (kBlock / kTile) * kTile) * kHead + lane * 16;
        const int8_t* k = c.codes[0] + from;
        const int8_t* v = c.codes[1] + from;
        const unsigned to = smem_u32(ring + stage * kStageBytes) + lane_token * kHead;
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i) {
          // chunk x of token t lies at x ^ (t % 8): no bank conflicts when fragments are read
          const unsigned off = to + i * 4 * kHead + ((lane_chunk ^ (i % 2 * 4 + lane_token)) << 4);
          if (i * 4 + lane_token < valid) {
            copy16(off, k + i * 4 * kHead);
            copy16(off + kTileBytes, v + i * 4 * kHead);
          }
        }
        // the next tile, its block's id one step ahead of its use
        if (--left > 0) {
          if (++tile == tiles) {
            tile = 0;
            if (++sub == lay.subs) {
              sub = 0;
              do {
                ++row;
                tiles = row_tiles(c, a, row);
              } while (tiles == 0);
              len = __ldg(a.row_len + row);
              table = c.table + (long long)__ldg(a.row_seq + row) * c.width;
            }
          }
          block = __ldg(table + tile / (kBlock / kTile));
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) load(s);

    unsigned qf[8][4];          // q in fragments: dims 32 q4 + 4 s + {0, 1 | 2, 3} of head g, high and low
    float qs = 0.0f;            // scale * log2(e) * the power of two that was taken out of q
    float m = 0.0f, l = 0.0f;   // head g: maximum (base 2) and this lane's share of the sum
    float o[16][2];             // head g: dims 32 q4 + j and 32 q4 + 16 + j
    bool whole = false;
    long long item = -1;
    int stage = 0;
    for (long long t = 0; t < todo; ++t) {
      copies_wait<kStages - 2>();
      __syncwarp();
      const Note note = notes[stage];
      if (note.item != item) {
        item = note.item;
        whole = note.flags & kFirst;
        const int it_row = (int)(item / lay.subs), it_sub = (int)(item % lay.subs);
        float4 q[8];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          q[s] = g < lay.count(it_sub) ? load4(static_cast<const T*>(a.q) + it_row * a.q_stride +
                                               (long long)(lay.first_q(it_sub) + g) * kHead + q4 * 32 + s * 4)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
          top = fmaxf(top, fmaxf(fmaxf(fabsf(q[s].x), fabsf(q[s].y)), fmaxf(fabsf(q[s].z), fabsf(q[s].w))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e and 2^e with the row's largest value in [1, 2) after the scaling
        const int e = top == 0.0f ? 127 : min(253, max(1, (int)(__float_as_uint(top) >> 23)));
        const float down = __uint_as_float((unsigned)(254 - e) << 23), up = __uint_as_float((unsigned)e << 23);
        qs = a.scale * up * 1.4426950408889634f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          split_half(q[s].x * down, q[s].y * down, qf[s][0], qf[s][1]);
          split_half(q[s].z * down, q[s].w * down, qf[s][2], qf[s][3]);
        }
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = 0.0f;
      }
      const uint8_t* kt = ring + stage * kStageBytes;
      const uint8_t* vt = kt + kTileBytes;
      const float ks = note.flags & kBad ? __int_as_float(0x7fc00000) : scales[stage * 2], vs = scales[stage * 2 + 1];

      // scores of tokens 8 j + 2 q4 + {0, 1}: the contraction may take the dims in any order, so a lane's 32
      // codes of token 8 j + g are two 16-byte chunks, four codes for each of the 8 steps
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
        const uint8_t* kr = kt + (j * 8 + g) * kHead;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 b = *reinterpret_cast<const uint4*>(kr + (((q4 * 2 + h) ^ g) << 4));
          const unsigned w[4] = {b.x ^ 0x80808080u, b.y ^ 0x80808080u, b.z ^ 0x80808080u, b.w ^ 0x80808080u};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mma(s[j], qf[h * 4 + i], codes_to_half2<0x5150>(w[i]), codes_to_half2<0x5352>(w[i]));
        }
      }
      const float cs = qs * ks;
      float p[4][2], tm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[j][i] = j * 8 + q4 * 2 + i < note.valid ? (s[j][i] + s[j][i + 2]) * cs : -INFINITY;
          tm = fmaxf(tm, p[j][i]);
        }
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
      float tl = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[j][i] = ex2(p[j][i] - tm);
          tl += p[j][i];
        }
      const float mn = fmaxf(m, tm), keep = ex2(m - mn), add = ex2(tm - mn), av = add * vs;
      m = mn;
      l = l * keep + add * tl;

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
        for (int i = 0; i < 4; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.0f;
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
          for (int i = 0; i < 4; ++i) mma(d[i], pf[k], b[0][i], b[1][i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[w * 4 + i][0] = fmaf(av, d[i][0] + d[i][2], o[w * 4 + i][0] * keep);
          o[w * 4 + i][1] = fmaf(av, d[i][1] + d[i][3], o[w * 4 + i][1] * keep);
        }
      }

      __syncwarp();  // the stage that is refilled next was read one step ago
      load((stage + kStages - 1) % kStages);
      stage = stage + 1 == kStages ? 0 : stage + 1;

      const bool ends = note.flags & kLast;
      if (ends || t == todo - 1) {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int it_sub = (int)(item % lay.subs);
        if (whole && ends) {
          if (g < lay.count(it_sub)) {
            const long long it_row = item / lay.subs;
            const int h = lay.first_q(it_sub) + g;
            const float r = 1.0f / l;
#pragma unroll
            for (int j = 0; j < 16; j += 4)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                put_out<T>(a, it_row, h, q4 * 32 + i * 16 + j, make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]), r);
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
          for (int j = 0; j < 16; j += 4)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *reinterpret_cast<float4*>(to + g * kHead + q4 * 32 + i * 16 + j) =
                  make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]);
          if (q4 == 0) {
            to[kRows * kHead + g] = m;
            to[kRows * kHead + kRows + g] = l;
          }
          if (lane == 0) {
            part_item[warp][whole] = item;
            if (!whole) part_ended[warp] = ends;
          }
        }
        item = -1;
      }
    }
    copies_wait<0>();
  }
  __syncthreads();

  // ---- join the warps' parts: part 2 w is warp w's item from before, part 2 w + 1 the one that goes on
  if (threadIdx.x < 2) info[2 * blockIdx.x + threadIdx.x] = -1;
  __syncthreads();
  auto part_at = [&](int p) {
    return p % 2 ? reinterpret_cast<const float*>(smem + p / 2 * kStages * kStageBytes)
                 : reinterpret_cast<const float*>(smem + kPartsOffset) + p / 2 * kPartFloats;
  };
  for (int first = 2 * warp; first < 2 * warp + 2; ++first) {
    const long long item = part_item[warp][first % 2];
    if (item < 0) continue;
    int prev = first - 1;
    while (prev >= 0 && part_item[prev / 2][prev % 2] < 0) --prev;
    if (prev >= 0 && part_item[prev / 2][prev % 2] == item) continue;  // joined by an earlier part's warp
    bool ended = first % 2 == 0 && part_ended[warp];
    int last = first;
    for (int p = first + 1; p < 2 * kWarps && !ended; ++p) {
      if (part_item[p / 2][p % 2] < 0) continue;
      if (part_item[p / 2][p % 2] != item) break;
      last = p;
      ended = p % 2 == 0 && part_ended[p / 2];
    }
    const int it_sub = (int)(item % lay.subs);
    const bool done = first % 2 == 1 && ended;
    const int slot = 2 * blockIdx.x + first % 2;
    for (int h = 0; h < lay.count(it_sub); ++h) {
      float m = -INFINITY, l = 0.0f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p = first; p <= last; ++p)
        if (part_item[p / 2][p % 2] == item) m = fmaxf(m, part_at(p)[kRows * kHead + h]);
      for (int p = first; p <= last; ++p) {
        if (part_item[p / 2][p % 2] != item) continue;
        const float* x = part_at(p);
        const float f = ex2(x[kRows * kHead + h] - m);
        const float4 v = *reinterpret_cast<const float4*>(x + h * kHead + lane * 4);
        l = fmaf(f, x[kRows * kHead + kRows + h], l);
        o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
      }
      if (done) {
        put_out<T>(a, item / lay.subs, lay.first_q(it_sub) + h, lane * 4, o, 1.0f / l);
        if (lane == 0) put_lse(a, item / lay.subs, lay.first_q(it_sub) + h, m, l);
      } else {
        float* to = work + (size_t)slot * kPartFloats;
        *reinterpret_cast<float4*>(to + h * kHead + lane * 4) = o;
        if (lane == 0) {
          to[kRows * kHead + h] = m;
          to[kRows * kHead + kRows + h] = l;
        }
      }
    }
    if (!done && lane == 0) info[slot] = first % 2 ? item : 2 * item + ended;
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
// on, head h of it. Four warps take every fourth part each, so that their loads overlap.
template <int kType>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(Cache c, Attend a) {
  using T = typename TypeOf<kType>::T;
  __shared__ float4 sum[kMergeThreads / 32][32];
  __shared__ float weight[kMergeThreads / 32], top[kMergeThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Layout lay(c, a);
  const float* work = static_cast<const float*>(a.work);
  const long long* info = reinterpret_cast<const long long*>(static_cast<const uint8_t*>(a.work) + kInfoOffset);
  const int cta = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long item = info[2 * cta + 1];
  if (item < 0 || h >= lay.count((int)(item % lay.subs))) return;
  // parts: 2 cta + 1, then the first ones of the CTAs behind up to the one where the item ends
  int n = 1;
  for (int base = cta + 1; base < kCtas; base += 32) {
    const long long x = base + lane < kCtas ? info[2 * (base + lane)] : -1;
    const unsigned end = __ballot_sync(0xffffffffu, x != 2 * item);  // ends there, or is another's
    n += end ? __ffs(end) - 1 : 32;
    if (end) {
      if (__shfl_sync(0xffffffffu, x, __ffs(end) - 1) == 2 * item + 1) ++n;
      break;
    }
  }
  auto part = [&](int i) { return work + (size_t)(i == 0 ? 2 * cta + 1 : 2 * (cta + i)) * kPartFloats; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < n; i += kMergeThreads) m = fmaxf(m, part(i)[kRows * kHead + h]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  if (lane == 0) top[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeThreads / 32; ++w) m = fmaxf(m, top[w]);
  float l = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = warp; i < n; i += kMergeThreads / 32) {
    const float* x = part(i);
    const float f = ex2(x[kRows * kHead + h] - m);
    const float4 v = *reinterpret_cast<const float4*>(x + h * kHead + lane * 4);
    l = fmaf(f, x[kRows * kHead + kRows + h], l);
    o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
  }
  sum[warp][lane] = o;
  if (lane == 0) weight[warp] = l;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < kMergeThreads / 32; ++w) {
    const float4 v = sum[w][lane];
    l += weight[w];
    o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
  }
  const int q_head = lay.first_q((int)(item % lay.subs)) + h;
  put_out<T>(a, item / lay.subs, q_head, lane * 4, o, 1.0f / l);
  if (lane == 0) put_lse(a, item / lay.subs, q_head, m, l);
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
