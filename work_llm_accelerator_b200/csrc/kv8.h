// 8-bit KV cache: blocks of 64 tokens, int8 codes with one fp32 scale per block and kv head, for K and for V
// (include/qwen_b200_ops.h has the layout and the definitions). Launchers of its kernels; arguments are
// checked by the entry points (ops_kv8.cu), indexes that live on the device by the kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace qb {
namespace kv8 {

constexpr int kBlock = 64;    // tokens of a block (the engine's page, kPage)
constexpr int kHead = 128;    // head dimension

struct Cache {
  int8_t* codes[2];    // K, V: [n_blocks][heads][64][128]
  float* scales[2];    // K, V: [n_blocks][heads]
  const int* table;    // [n_seqs][width] block ids
  int n_blocks, heads, n_seqs, width;
};

// Rows of a call: segment i is rows offsets[i] .. offsets[i + 1] - 1 = positions starts[i] .. of sequence seqs[i].
struct Rows {
  const int *seqs, *starts, *offsets;
  int segments;
  long long n_rows;  // rows that the buffers hold
  long long stride;  // elements from row to row
};

// `type`: 0 fp32, 1 fp16, 2 bf16.
cudaError_t launch_append(const Cache& c, const void* k, const void* v, int type, const Rows& r, cudaStream_t s);
cudaError_t launch_read(const Cache& c, void* k, void* v, int type, const Rows& r, cudaStream_t s);

struct Attend {
  const void* q;
  void* out;
  float* lse;  // may be null
  long long q_stride, out_stride;
  const int *row_seq, *row_len;
  int rows, q_heads;
  float scale;
  void* work;
};
size_t attention_workspace(int rows, int q_heads, int heads);  // the same for all: it follows from the number of CTAs
cudaError_t launch_attention(const Cache& c, const Attend& a, int type, cudaStream_t s);

// Error flags of the kernels on the current device (kErrMbarTimeout, kErrBadIndex).
unsigned kernel_error(bool reset);
unsigned attention_kernel_error(bool reset);

}  // namespace kv8
}  // namespace qb
