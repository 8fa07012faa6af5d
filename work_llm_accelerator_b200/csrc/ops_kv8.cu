// Entry points of the 8-bit KV cache operators and of token sampling (include/qwen_b200_ops.h): the argument
// checks that the host can make, then one launch on the caller's stream. Nothing here allocates or synchronises,
// so every call can be captured into a graph.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/qwen_b200_ops.h"
#include "kv8.h"
#include "qwen_kernels.cuh"
#include "runtime.h"
#include "sample.h"

namespace qb {
namespace {

constexpr long long kMaxRows = 1 << 24;

struct Arg {
  const char* name;
  const void* p;
  int align;
};

bool range_ok(const char* op, const char* name, long long v, long long lo, long long hi) {
  if (v >= lo && v <= hi) return true;
  set_error("%s: %s is %lld, outside %lld..%lld", op, name, v, lo, hi);
  return false;
}

// Memory of device `dev`, or managed memory. The driver's own query takes half of the runtime's time, and a call asks for
// up to eleven buffers; where it cannot be had, the runtime answers.
bool on_device(const void* p, int dev) {
  static const PFN_cuPointerGetAttributes_v7000 query = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    return cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &r) == cudaSuccess &&
                   r == cudaDriverEntryPointSuccess
               ? reinterpret_cast<PFN_cuPointerGetAttributes_v7000>(f)
               : nullptr;
  }();
  if (query) {
    unsigned type = 0, managed = 0;  // a type of 0: not known to CUDA
    int ordinal = -1;
    CUpointer_attribute names[3] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                    CU_POINTER_ATTRIBUTE_IS_MANAGED};
    void* values[3] = {&type, &ordinal, &managed};
    return query(3, names, values, reinterpret_cast<CUdeviceptr>(p)) == CUDA_SUCCESS &&
           (managed || (type == CU_MEMORYTYPE_DEVICE && ordinal == dev));
  }
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev);
}

// Every buffer: present, aligned, and memory of the current device (or managed memory).
int check_buffers(const char* op, const Arg* args, int n) {
  for (int i = 0; i < n; ++i) {
    if (!args[i].p) {
      set_error("%s: %s is null", op, args[i].name);
      return kStatusInvalid;
    }
    if (reinterpret_cast<uintptr_t>(args[i].p) % args[i].align) {
      set_error("%s: %s is not %d-byte aligned", op, args[i].name, args[i].align);
      return kStatusInvalid;
    }
  }
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    set_error("%s: no current CUDA device", op);
    return kStatusNoDevice;
  }
  for (int i = 0; i < n; ++i) {
    if (!on_device(args[i].p, dev)) {
      set_error("%s: %s must be memory of the current device (%d) or managed memory", op, args[i].name, dev);
      return kStatusInvalid;
    }
  }
  return 0;
}

bool cache_ok(const char* op, const qwen_b200_kv8_cache* c) {
  if (!c) {
    set_error("%s: cache is null", op);
    return false;
  }
  return range_ok(op, "n_blocks", c->n_blocks, 1, INT32_MAX) && range_ok(op, "n_kv_heads", c->n_kv_heads, 1, 1024) &&
         range_ok(op, "n_blocks * n_kv_heads", (long long)c->n_blocks * c->n_kv_heads, 1, INT32_MAX) &&
         range_ok(op, "n_seqs", c->n_seqs, 1, INT32_MAX) &&
         range_ok(op, "max_blocks", c->max_blocks, 1, INT32_MAX / kv8::kBlock);
}

kv8::Cache view(const qwen_b200_kv8_cache* c) {
  kv8::Cache v;
  v.codes[0] = reinterpret_cast<int8_t*>(c->k_codes);
  v.codes[1] = reinterpret_cast<int8_t*>(c->v_codes);
  v.scales[0] = c->k_scales;
  v.scales[1] = c->v_scales;
  v.table = c->block_table;
  v.n_blocks = c->n_blocks;
  v.heads = c->n_kv_heads;
  v.n_seqs = c->n_seqs;
  v.width = c->max_blocks;
  return v;
}

int size_of(int dtype) { return dtype == QWEN_B200_F32 ? 4 : 2; }

bool stride_ok(const char* op, const char* name, long long stride, long long least, int dtype) {
  if (stride >= least && stride <= (1ll << 40) && stride * size_of(dtype) % 16 == 0) return true;
  set_error("%s: %s %lld must be at least %lld elements and a multiple of 16 bytes", op, name, stride, least);
  return false;
}

int done(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return 0;
  set_error("%s: %s", op, cudaGetErrorString(e));
  return kStatusCuda;
}

// Writing and reading back take the same arguments.
template <bool kWrite>
int rows_call(const char* op, const qwen_b200_kv8_cache* c, const void* k, const void* v, int dtype, long long row_stride,
              long long n_rows, const int* seqs, const int* starts, const int* offsets, int n_segments, void* stream) {
  if (!cache_ok(op, c) || !range_ok(op, "dtype", dtype, QWEN_B200_F32, QWEN_B200_BF16) ||
      !range_ok(op, "n_rows", n_rows, 0, kMaxRows) || !range_ok(op, "n_segments", n_segments, 0, kMaxRows) ||
      !stride_ok(op, "row_stride", row_stride, (long long)c->n_kv_heads * kv8::kHead, dtype))
    return kStatusInvalid;
  if (n_rows == 0 || n_segments == 0) return 0;
  if (!kWrite && k == v && k) {
    set_error("%s: k and v are one buffer", op);
    return kStatusInvalid;
  }
  const Arg args[] = {{"k", k, 16},
                      {"v", v, 16},
                      {"k_codes", c->k_codes, 16},
                      {"v_codes", c->v_codes, 16},
                      {"k_scales", c->k_scales, 4},
                      {"v_scales", c->v_scales, 4},
                      {"block_table", c->block_table, 4},
                      {"seqs", seqs, 4},
                      {"starts", starts, 4},
                      {"offsets", offsets, 4}};
  if (const int st = check_buffers(op, args, 10)) return st;
  const kv8::Rows r{seqs, starts, offsets, n_segments, n_rows, row_stride};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kWrite) return done(op, kv8::launch_append(view(c), k, v, dtype, r, s));
  return done(op, kv8::launch_read(view(c), const_cast<void*>(k), const_cast<void*>(v), dtype, r, s));
}

}  // namespace
}  // namespace qb

extern "C" int qwen_b200_kv8_append(const qwen_b200_kv8_cache* cache, const void* k, const void* v, int dtype,
                                    long long row_stride, long long n_rows, const int* seqs, const int* starts,
                                    const int* offsets, int n_segments, void* stream) {
  return qb::rows_call<true>("qwen_b200_kv8_append", cache, k, v, dtype, row_stride, n_rows, seqs, starts, offsets,
                             n_segments, stream);
}

extern "C" int qwen_b200_kv8_read(const qwen_b200_kv8_cache* cache, void* k, void* v, int dtype, long long row_stride,
                                  long long n_rows, const int* seqs, const int* starts, const int* offsets,
                                  int n_segments, void* stream) {
  return qb::rows_call<false>("qwen_b200_kv8_read", cache, k, v, dtype, row_stride, n_rows, seqs, starts, offsets,
                              n_segments, stream);
}

extern "C" long long qwen_b200_kv8_attention_workspace(int n_rows, int n_q_heads, int n_kv_heads) {
  using namespace qb;
  const char* op = "qwen_b200_kv8_attention_workspace";
  if (!range_ok(op, "n_rows", n_rows, 0, 1 << 20) || !range_ok(op, "n_kv_heads", n_kv_heads, 1, 1024) ||
      !range_ok(op, "n_q_heads", n_q_heads, 1, 1024))
    return -1;
  return (long long)kv8::attention_workspace(n_rows, n_q_heads, n_kv_heads);
}

extern "C" int qwen_b200_kv8_attention(const qwen_b200_kv8_cache* cache, const void* q, long long q_stride, void* out,
                                       long long out_stride, int dtype, int n_rows, int n_q_heads, const int* row_seqs,
                                       const int* row_lens, float scale, void* workspace, long long workspace_bytes,
                                       float* lse, void* stream) {
  using namespace qb;
  const char* op = "qwen_b200_kv8_attention";
  if (!cache_ok(op, cache) || !range_ok(op, "dtype", dtype, QWEN_B200_F32, QWEN_B200_BF16) ||
      !range_ok(op, "n_rows", n_rows, 0, 1 << 20) || !range_ok(op, "n_q_heads", n_q_heads, 1, 1024) ||
      !stride_ok(op, "q_stride", q_stride, (long long)n_q_heads * kv8::kHead, dtype) ||
      !stride_ok(op, "out_stride", out_stride, (long long)n_q_heads * kv8::kHead, dtype))
    return kStatusInvalid;
  if (n_q_heads % cache->n_kv_heads) {
    set_error("%s: n_q_heads %d is not a multiple of n_kv_heads %d", op, n_q_heads, cache->n_kv_heads);
    return kStatusInvalid;
  }
  // items, a row's tiles and a CTA's share of all tiles are counted in 31 bits
  if (!range_ok(op, "n_q_heads * max_blocks", (long long)n_q_heads * cache->max_blocks, 0, 1ll << 29) ||
      !range_ok(op, "n_rows * n_q_heads", (long long)n_rows * n_q_heads, 0, 1ll << 29) ||
      !range_ok(op, "n_rows * n_q_heads * max_blocks", (long long)n_rows * n_q_heads * cache->max_blocks, 0, 1ll << 36))
    return kStatusInvalid;
  if (!std::isfinite(scale)) {
    set_error("%s: scale is not finite", op);
    return kStatusInvalid;
  }
  if (n_rows == 0) return 0;
  const long long need = (long long)kv8::attention_workspace(n_rows, n_q_heads, cache->n_kv_heads);
  if (workspace_bytes < need) {
    set_error("%s: workspace of %lld bytes, %lld needed", op, workspace_bytes, need);
    return kStatusInvalid;
  }
  if (q == out && q) {
    set_error("%s: out is q; they must not overlap", op);
    return kStatusInvalid;
  }
  const Arg args[] = {{"q", q, 16},
                      {"out", out, 16},
                      {"k_codes", cache->k_codes, 16},
                      {"v_codes", cache->v_codes, 16},
                      {"k_scales", cache->k_scales, 4},
                      {"v_scales", cache->v_scales, 4},
                      {"block_table", cache->block_table, 4},
                      {"row_seqs", row_seqs, 4},
                      {"row_lens", row_lens, 4},
                      {"workspace", workspace, 16},
                      {"lse", lse, 4}};
  if (const int st = check_buffers(op, args, lse ? 11 : 10)) return st;
  const kv8::Attend a{q, out, lse, q_stride, out_stride, row_seqs, row_lens, n_rows, n_q_heads, scale, workspace};
  return done(op, kv8::launch_attention(view(cache), a, dtype, static_cast<cudaStream_t>(stream)));
}

extern "C" int qwen_b200_sample(const void* logits, int dtype, int rows, int vocab, long long row_stride,
                                const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                                const float* uniforms, int* tokens, float* probs, void* stream) {
  using namespace qb;
  const char* op = "qwen_b200_sample";
  if (!range_ok(op, "dtype", dtype, QWEN_B200_F32, QWEN_B200_BF16) || !range_ok(op, "rows", rows, 0, 1 << 20) ||
      !range_ok(op, "vocab", vocab, 1, sampling::kMaxVocab) || !range_ok(op, "row_stride", row_stride, vocab, 1ll << 40))
    return kStatusInvalid;
  if (rows == 0) return 0;
  Arg args[8] = {{"logits", logits, size_of(dtype)}, {"uniforms", uniforms, 4}, {"tokens", tokens, 4}};
  int n = 3;
  if (temperature) args[n++] = {"temperature", temperature, 4};
  if (top_k) args[n++] = {"top_k", top_k, 4};
  if (top_p) args[n++] = {"top_p", top_p, 4};
  if (min_p) args[n++] = {"min_p", min_p, 4};
  if (probs) args[n++] = {"probs", probs, 4};
  if (const int st = check_buffers(op, args, n)) return st;
  const sampling::Sample a{logits, rows, vocab, row_stride, temperature, top_k, top_p, min_p, uniforms, tokens, probs};
  return done(op, sampling::launch_sample(a, dtype, static_cast<cudaStream_t>(stream)));
}
