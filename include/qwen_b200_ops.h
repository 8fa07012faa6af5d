/*
 * Device-pointer operator API of libqwen_b200.so: single hot-path kernels on buffers the caller already
 * holds in GPU memory, enqueued on the caller's stream (no host staging, no synchronisation).
 * Status codes: 0 ok, 1 invalid argument (message in qwen_b200_last_error()), 30 CUDA failure.
 */
#ifndef QWEN_B200_OPS_H
#define QWEN_B200_OPS_H

#ifdef __cplusplus
extern "C" {
#endif

/* Decode attention context for one token: 12 query heads over 2 KV heads, head_dim 128 (replaces the
 * reference's decode_attention_context, hls/decode_only/qwen_decode_attention_kernel.cpp:113-162).
 *   q        [1536] fp32, the token's post-RoPE query (device memory)
 *   k_cache  [seq_len][256] fp32 token-major keys (device memory), the token's own row included
 *   v_cache  [seq_len][256] fp32 token-major values (device memory)
 *   context  [1536] fp32 output (device memory)
 *   stream   cudaStream_t (NULL = legacy default stream)
 * The split-history scratch is allocated by the library on a device's first call and grown when a
 * longer history arrives; calls on one device share it, so calls that overlap on the GPU race. */
int qwen_b200_decode_attention(const float* q, const float* k_cache, const float* v_cache, int seq_len,
                               float* context, void* stream);

/* Same computation and arguments as qwen_b200_decode_attention, for callers that cannot allocate device
 * memory at the point where they run attention -- e.g. a serving runtime that reserves all GPU memory in
 * its own pool at start-up, or a latency-critical loop where cudaMalloc/cudaFree would synchronise the
 * device. No counterpart in the reference (its host library has no device memory at all). It allocates
 * nothing: its scratch is a fixed array compiled into the library (about 0.8 MB, held on every GPU that
 * loads the library until the process exits), so seq_len is limited to 8192 (status 1 above it). The
 * first call on a device looks up that array's address and should come before any stream capture. All
 * calls on a device share the array (each call clears the parts that must start at zero), so calls that
 * overlap on the GPU race. */
int qwen_b200_decode_attention_noalloc(const float* q, const float* k_cache, const float* v_cache, int seq_len,
                                       float* context, void* stream);

/* Integer core of the W8 projections on the int8 tensor cores, exposed so that its exactness can be
 * checked: the fp32 activations x[t] (t < n_tokens <= 4, length k) are written as step[t] * X with
 * step[t] = max|x[t]| / 8355710 (fp32 division; 1.0 for an all-zero row) and X = rint(x / step) split into
 * balanced int8 digits X = d0 + 256 d1 + 65536 d2, each in [-128, 127]; then
 *   acc[r][4 d + t] = sum_i codes[r][i] * d_d(t, i)     (int32, exact)
 * for every row r, and 0 in the columns of absent tokens. The W8 projections compute
 * y = scale[r] * step[t] * (acc0 + 256 acc1 + 65536 acc2) from the same sums, in place of the reference's
 * fp32 dot product (hls/decode_only/qwen_decode_attention_kernel.cpp:62-98).
 *   codes  [rows][k] int8 weight codes (device memory, 16-byte aligned), rows % 128 == 0, k % 128 == 0
 *   x      [n_tokens][k] fp32 (device memory)
 *   acc    [rows][12] int32 output (device memory);  step  [n_tokens] fp32 output (device memory) */
int qwen_b200_w8_digit_products(const signed char* codes, int rows, int k, const float* x, int n_tokens, int* acc,
                                float* step, void* stream);

/* Many-token form of the same integer core (the prefill and batched projections): x [n_tokens][k] fp32
 * (16-byte aligned) becomes three digit planes with the per-token step as above, and
 *   acc[d][t][r] = sum_i codes[r][i] * d_d(t, i)      (int32, exact), d < 3, t < n_tokens, r < rows
 * acc is [3][n_tokens][rows] int32, step [n_tokens] fp32 (device memory). Uses stream-ordered temporary
 * allocations for the planes. rows % 128 == 0, k % 128 == 0, 1 <= n_tokens <= 65536. */
int qwen_b200_w8_digit_planes(const signed char* codes, int rows, int k, const float* x, int n_tokens, int* acc,
                              float* step, void* stream);

/* Causal prefill attention context of seq_len tokens (replaces the reference's two-pass prefill context,
 * hls/prefill_only/qwen_prefill_attention_kernel.cpp:204-289): for every query t and head h,
 *   max = max_{j<=t} s_j,  e_j = approx_exp(s_j - max),  context = (sum_j e_j v_j) * (1 / sum_j e_j)
 * with s_j = (q_h . k_j) * 0.08838834764831845 and the reference's approx_exp.
 *   q        [seq_len][1536] fp32 post-RoPE queries (device memory, 16-byte aligned)
 *   k_cache  [seq_len][256] fp32 token-major keys (device memory, 16-byte aligned)
 *   v_cache  [seq_len][256] fp32 token-major values (device memory)
 *   context  [seq_len][1536] fp32 output (device memory, 16-byte aligned)
 *   mode     0: tensor cores (operands as fp16 hi + lo pairs, fp32 accumulation; inputs with |x| >= 32768
 *               or non-finite values are computed by the CUDA-core kernel instead), 1: CUDA cores (fp32)
 * Mode 0 uses stream-ordered temporary allocations (about 8 KB per token). */
int qwen_b200_prefill_attention(const float* q, const float* k_cache, const float* v_cache, int seq_len,
                                float* context, int mode, void* stream);

/* The prefill softmax exponential as the tensor-core attention evaluates it: y[i] = approx_exp(x[i])
 * (hls/prefill_only/qwen_prefill_attention_kernel.cpp:47-110, degree-6 Taylor series with halving and
 * squaring), evaluated without divisions or branches; exposed so that its bit-identity with the reference's
 * function can be checked.
 * x, y [n] fp32 device memory. */
int qwen_b200_prefill_approx_exp(const float* x, float* y, long long n, void* stream);

/* The decode softmax and SiLU exponential of the engine's "exact" option: y[i] = expf(x[i]) exactly as the
 * reference host library's expf computes it (hls/decode_only/qwen_decode_attention_kernel.cpp:149 and
 * qwen_decode_mlp_kernel.cpp:80 call std::exp on floats, which resolves to glibc's expf: a 32-entry 2^(i/32)
 * table and a degree-3 polynomial in double, restated with the fused multiply-adds of glibc's x86-64 FMA
 * build). Exposed so that its identity with the host C library can be checked.
 * x, y [n] fp32 device memory. */
int qwen_b200_exact_expf(const float* x, float* y, long long n, void* stream);

/* Element types of the operators below. Whatever the type, they compute in fp32 or, as said there, in integers of about as
 * many bits, and round results once. */
enum { QWEN_B200_F32 = 0, QWEN_B200_F16 = 1, QWEN_B200_BF16 = 2 };

/* An 8-bit KV cache of one layer, in buffers of the caller (device memory): blocks of 64 tokens, head dimension
 * 128, int8 codes, one fp32 scale per block and kv head; a cached value is code * scale. No counterpart in the
 * reference, whose caches are fp32 (hls/common/llm_memory_layout.h).
 *   k_codes, v_codes    [n_blocks][n_kv_heads][64][128] int8 (16-byte aligned)
 *   k_scales, v_scales  [n_blocks][n_kv_heads] fp32
 *   block_table         [n_seqs][max_blocks] int32: token t of sequence s is slot t % 64 of block
 *                       block_table[s][t / 64]; entries behind a sequence's last block are not read
 * Blocks need no initialisation. Indexes that live on the device are checked there; a kernel that meets one outside of
 * its buffers touches nothing there and sets bit 1 of qwen_b200_kernel_error(): a block id reads as NaN and is not
 * written, a segment whose sequence, positions or rows lie outside is left out, and an attention row whose sequence or
 * length does is NaN. */
typedef struct qwen_b200_kv8_cache {
  signed char* k_codes;
  signed char* v_codes;
  float* k_scales;
  float* v_scales;
  int n_blocks;
  int n_kv_heads;
  const int* block_table;
  int n_seqs;
  int max_blocks;
} qwen_b200_kv8_cache;

/* Write K and V rows into the cache (each row: n_kv_heads x 128 values, row_stride elements apart, so that rows may
 * lie inside q|k|v rows). Segment i appends rows offsets[i] .. offsets[i + 1] - 1 to sequence seqs[i], which holds
 * starts[i] tokens already; offsets [n_segments + 1] ascend from 0, equal ones make an empty segment, and rows from
 * offsets[n_segments] to n_rows (a padded batch) are ignored. Per kv head, for K and for V:
 *   a block that the call opens (its first new slot is slot 0) gets scale = max|x| * fl(1 / 127), at least 2^-126 (0
 *   if every value is 0); a block with earlier tokens keeps its scale, doubled as often as needed to reach that value,
 *   and the codes of its earlier tokens are halved as often; code = clamp(rint(x / scale), -127, 127), ties to even.
 * A value written with its whole block is off by at most scale / 2, one that was halved later by less than scale.
 * Appending again from an earlier position (a dropped draft) overwrites. A NaN or an infinity makes its block's scale
 * NaN: the block reads as NaN until it is opened again.
 * A block shared by several sequences must not be written, and a call must not name a sequence twice (the values of
 * such blocks would be undefined, with no access out of bounds).
 *   k, v                  [n_rows] rows of `dtype` (16-byte aligned; row_stride a multiple of 16 bytes)
 *   seqs, starts, offsets [n_segments], [n_segments], [n_segments + 1] int32 (device memory) */
int qwen_b200_kv8_append(const qwen_b200_kv8_cache* cache, const void* k, const void* v, int dtype,
                         long long row_stride, long long n_rows, const int* seqs, const int* starts,
                         const int* offsets, int n_segments, void* stream);

/* Read cached rows back: segment i writes tokens starts[i] .. of sequence seqs[i] to rows offsets[i] ..
 * offsets[i + 1] - 1 of k and v (different buffers), as code * scale rounded to `dtype` (a value within 1% of the
 * type's largest number can lie beyond it by then, and reads as infinity). Arguments as above; rows from
 * offsets[n_segments] on are left as they are, and a sequence may be named more than once. */
int qwen_b200_kv8_read(const qwen_b200_kv8_cache* cache, void* k, void* v, int dtype, long long row_stride,
                       long long n_rows, const int* seqs, const int* starts, const int* offsets, int n_segments,
                       void* stream);

/* Decode attention over the 8-bit cache, one query row per new token (replaces the context of
 * hls/decode_only/qwen_decode_attention_kernel.cpp:113-162 for a cache in this form). Row r of sequence
 * row_seqs[r] attends to the sequence's first row_lens[r] tokens (its own included: append first); drafted tokens of
 * one sequence are rows with lengths that rise by one. Query head h reads kv head h / (n_q_heads / n_kv_heads).
 *   s_j = scale * (q . k_j),  out = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
 * Both products are sums of integers: a query head is held to 2^-30 of its largest channel, and a weight to 2^-30 of the
 * largest of the up to 32 tokens that it is computed with, in place of 2^-24 of itself; the sums are exact, and what
 * follows is fp32.
 * A call repeats bit for bit. How a row's tokens are split into parts follows from the lengths of all rows, so the same row
 * in another batch, or at another place, may differ by the roundings of its sums.
 * row_lens[r] == 0: out is 0 and lse -infinity. row_seqs[r] < 0 (a padded row): out and lse are left as they are.
 *   q, out     [n_rows] rows of n_q_heads x 128 values of `dtype` (16-byte aligned, strides in elements, multiples
 *              of 16 bytes); out must not overlap q
 *   row_seqs, row_lens  [n_rows] int32 (device memory)
 *   workspace  at least qwen_b200_kv8_attention_workspace(n_rows, n_q_heads, n_kv_heads) bytes of device memory
 *              (16-byte aligned, any contents); calls that overlap on the GPU need one each
 *   lse        [n_rows][n_q_heads] fp32, or NULL */
int qwen_b200_kv8_attention(const qwen_b200_kv8_cache* cache, const void* q, long long q_stride, void* out,
                            long long out_stride, int dtype, int n_rows, int n_q_heads, const int* row_seqs,
                            const int* row_lens, float scale, void* workspace, long long workspace_bytes, float* lse,
                            void* stream);
/* Bytes of that workspace, -1 for an argument out of range. */
long long qwen_b200_kv8_attention_workspace(int n_rows, int n_q_heads, int n_kv_heads);

/* Sample one token per row from its logits and a given uniform number (the reference only takes the argmax,
 * verification/real_host_top_backend.py:138-146). With the row's tokens sorted by logit (ties: lowest index first),
 * w_i = exp((logit_i - max) / temperature):
 *   top_k > 0  keeps the first top_k;
 *   top_p < 1  keeps the fewest of those, at least one, whose sum of w reaches top_p of their whole sum;
 *   min_p > 0  keeps those of w >= min_p (the first one in any case);
 * the token is the first whose running sum of w exceeds uniform * (sum of the kept w), the last one kept if none does.
 * temperature below 2^-126 (0 included) or NaN: the first token, with probability 1; one from there to 2^-121 counts as
 * 2^-121. Logits of -infinity or NaN are
 * never taken; a row without any other gives token -1, probability 0. +infinity outweighs every finite logit. Weights
 * below exp(-32) of the largest count as 0; the others are within (2 + z) 2^-24 of themselves, z = (max - logit) /
 * temperature; a logit whose distance from the largest is beyond the fp32 range counts as -infinity.
 *   logits      [rows][vocab] of `dtype`, rows row_stride elements apart; 1 <= vocab <= 262144
 *   temperature, top_k, top_p, min_p  [rows] fp32 / int32, or NULL (1, off, off, off)
 *   uniforms    [rows] fp32 in [0, 1); below (or NaN) counts as 0, above draws the last token kept
 *   tokens      [rows] int32;  probs  [rows] fp32: the probability that the token had among the kept ones, or NULL
 * All device memory. The result does not depend on the order in which anything is summed on the GPU. */
int qwen_b200_sample(const void* logits, int dtype, int rows, int vocab, long long row_stride, const float* temperature,
                     const int* top_k, const float* top_p, const float* min_p, const float* uniforms, int* tokens,
                     float* probs, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QWEN_B200_OPS_H */
