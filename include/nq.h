/*
 * nq.h -- C ABI of the B200 quantized-matmul library (libnq.so).
 *
 * The entry points replace the quantized-linear calls that neurons' models
 * make into MLX (MLXBackend serves them today):
 *   nq_quantized_matmul  <- mx::quantized_matmul(x, w, scales, biases,
 *                           transpose=true, gs, bits, "affine")
 *                           compute/src/compute/model/mlx_ops.h:28-42 (lin)
 *   nq_dequantize        <- mx::dequantize(w, scales, biases, gs, bits)
 *                           compute/src/compute/model/llama_model.cpp:67,
 *                           gemma_model_mlx.cpp:82, qwen3_moe_model_mlx.cpp:411,
 *                           qwen3_transformer_moe_model_mlx.cpp:183
 *   nq_gather_qmm        <- mx::gather_qmm(x, w, scales, biases, lhs=nullopt,
 *                           rhs=topk_idx, transpose=true, gs, bits)
 *                           qwen3_transformer_moe_model_mlx.cpp:69-74,
 *                           qwen3_moe_model_mlx.cpp:356-364
 *   nq_moe_route         <- router of the switch step (softmax fp32, top-k,
 *                           renormalise) qwen3_transformer_moe_model_mlx.cpp:36-48
 *   nq_moe_switch        <- the whole switch-MLP step for T tokens
 *                           (gate/up gather_qmm, SwiGLU, down gather_qmm,
 *                           score-weighted sum) qwen3_transformer_moe_model_mlx.cpp:29-79;
 *                           batched over tokens instead of the token loop at
 *                           qwen3_transformer_moe_model_mlx.cpp:479-486
 *   nq_quantize          <- mx::quantize(w, gs, bits) (MLX affine; the
 *                           reference loads pre-quantized checkpoints and has
 *                           no call site of its own)
 *   nq_paged_*, nq_pages_*  the key/value cache in pages: attention of new
 *                           tokens over it, the append, and the page pool (no
 *                           counterpart: the reference's caches grow by
 *                           concatenation, llama_model.cpp:462-463)
 *   nq_bits_from_shapes  <- mlx_ops::bits  compute/src/compute/model/mlx_ops.h:20-25
 *
 * Conventions
 *   - Every tensor pointer is a DEVICE pointer (cudaMalloc'd or equivalent),
 *     row-major and contiguous.  bf16 tensors are passed as uint16_t bit
 *     patterns.  Packed weights are uint32 words holding 32/bits codes, the
 *     lowest-index code in the lowest bits (MLX layout).
 *   - Weight shapes follow MLX's transpose=true layout: w [N, K*bits/32],
 *     scales and biases [N, K/group_size]; stacked experts prepend [E].
 *   - bits is 4 or 8; group_size is 32, 64 or 128; K % group_size == 0.
 *   - stream is a cudaStream_t (NULL = the legacy default stream).  Every call
 *     is asynchronous on that stream and allocates nothing.
 *   - Return value: an nq_status.  The message of the last failure on the
 *     calling thread is available from nq_last_error().
 */
#ifndef NQ_H_
#define NQ_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Mirrors compute::ErrorCode (compute/src/compute/core/compute_types.h:9-16). */
typedef enum nq_status {
    NQ_SUCCESS = 0,
    NQ_INVALID_INPUT = 1,
    NQ_INVALID_MODEL = 2,
    NQ_BACKEND_NOT_AVAILABLE = 3,
    NQ_COMPUTE_ERROR = 4,
    NQ_UNKNOWN_ERROR = 5
} nq_status;

/* Quantization schemes for nq_quantize. */
#define NQ_SCHEME_MLX_AFFINE 0 /* MLX affine quantizer (edge snapping) */
#define NQ_SCHEME_MINMAX 1     /* scale=(max-min)/(2^bits-1), bias=min */

/* Input dtypes for nq_quantize. */
#define NQ_DTYPE_F32 0
#define NQ_DTYPE_BF16 1
#define NQ_DTYPE_F16 2

/* Library identity / diagnostics (no reference counterpart: FFI plumbing). */
int nq_version(void);
const char *nq_last_error(void);
/* Number of CUDA devices usable by the library (0 when none); never fails. */
int nq_device_count(void);
/* Reads and clears the device-side error word of the current device: bit 0, a
 * kernel's bounded wait ran out; bit 1, an index that a kernel read was out of
 * range (gather index, token, table row, length, page); bit 2, a page request
 * was refused (nq_pages_*).  0 = no error. */
int nq_take_device_error(unsigned int *err_out);

/* mlx_ops::bits: round(32 * (w_cols / s_cols) / group_size), 4 if not positive. */
int nq_bits_from_shapes(int64_t w_cols, int64_t s_cols, int group_size);

/* mx::quantize.  w: [rows, K] fp32, bf16 or fp16 (w_dtype).  Outputs: wq
 * [rows, K*bits/32] uint32, scales/biases [rows, K/group_size] bf16 (fp16 for
 * fp16 weights: MLX keeps the weights' dtype). */
int nq_quantize(const void *w, int w_dtype, int64_t rows, int64_t K, int bits,
                int group_size, int scheme, uint32_t *wq, uint16_t *scales,
                uint16_t *biases, void *stream);

/* mx::dequantize.  out: [rows, K] bf16, bit-exact bf16(bf16(s*q) + b). */
int nq_dequantize(const uint32_t *wq, const uint16_t *scales,
                  const uint16_t *biases, int64_t rows, int64_t K, int bits,
                  int group_size, uint16_t *out, void *stream);

/* mx::dequantize with fp16 scales and biases (an fp16 checkpoint): out
 * [rows, K] fp16, bit-exact fp16(fp16(s*q) + b). */
int nq_dequantize_f16(const uint32_t *wq, const uint16_t *scales,
                      const uint16_t *biases, int64_t rows, int64_t K, int bits,
                      int group_size, uint16_t *out, void *stream);

/* mx::quantized_matmul with fp16 x, scales, biases and y (what mlx_ops::lin,
 * compute/src/compute/model/mlx_ops.h:33-39, runs for an fp16 checkpoint):
 * fp32 accumulation, fp16 out.  M <= 8 with 4-bit codes takes the decode
 * GEMV (K % 128 == 0, at most 96 KB of x); every other shape the tcgen05
 * GEMM (16-byte aligned x and packed rows). */
int nq_quantized_matmul_f16(const uint16_t *x, int64_t M, const uint32_t *wq,
                            const uint16_t *scales, const uint16_t *biases,
                            int64_t N, int64_t K, int bits, int group_size,
                            uint16_t *y, void *stream);

/* mx::quantized_matmul(x, w, scales, biases, transpose=true, gs, bits).
 * x: [M, K] bf16; y: [M, N] bf16.  fp32 accumulation.  biases must be
 * non-NULL (affine mode).  M may be 0. */
int nq_quantized_matmul(const uint16_t *x, int64_t M, const uint32_t *wq,
                        const uint16_t *scales, const uint16_t *biases,
                        int64_t N, int64_t K, int bits, int group_size,
                        uint16_t *y, void *stream);

/* Number of kernels one nq_quantized_matmul call of this shape launches on the
 * current device (no reference counterpart: profiling aid).  1 for the GEMV
 * and for most tensor-core problems; 2 when the tensor-core grid's last wave
 * is split along K (a clustered tail kernel, then the whole tiles); 0 for
 * M == 0 or N == 0; a negative status for invalid arguments. */
int nq_quantized_matmul_launches(int64_t M, int64_t N, int64_t K, int bits, int group_size);

/* mx::gather_qmm(x, w, scales, biases, lhs_indices, rhs_indices,
 * transpose=true, gs, bits).
 *   x: [x_batch, M, K] bf16;  w: [E, N, K*bits/32];  scales/biases [E, N, K/gs]
 *   out[i] ([M, N] slice of y: [n_idx, M, N]) = x[xi] . dequant(w[rhs[i]])^T,
 *   xi = lhs[i] when lhs_indices != NULL, else i when x_batch == n_idx, else 0
 *   (x_batch == 1 broadcasts).  Index arrays are DEVICE int32 arrays; indices
 *   out of range make the affected output rows zero and raise the device error
 *   word (nq_take_device_error). */
int nq_gather_qmm(const uint16_t *x, int64_t x_batch, int64_t M,
                  const int32_t *lhs_indices, const int32_t *rhs_indices,
                  int64_t n_idx, const uint32_t *wq, const uint16_t *scales,
                  const uint16_t *biases, int64_t E, int64_t N, int64_t K,
                  int bits, int group_size, uint16_t *y, void *stream);

/* Router of the MoE switch step.  logits: [T, E] bf16 (the output of the
 * router linear).  Outputs topk_idx [T, top_k] int32 (descending probability,
 * ties -> lower expert index) and topk_scores [T, top_k] fp32 (softmax over
 * all E experts, renormalised over the selected top_k).  top_k <= 32,
 * E <= 1024. */
int nq_moe_route(const uint16_t *logits, int64_t T, int64_t E, int64_t top_k,
                 int32_t *topk_idx, float *topk_scores, void *stream);

/* Workspace bytes nq_moe_switch needs for T tokens. */
size_t nq_moe_workspace_size(int64_t T, int64_t E, int64_t top_k, int64_t H,
                             int64_t I);

/* Switch-MLP of one MoE layer for T tokens (batched over tokens):
 *   y[t] = sum_j bf16(score[t,j]) * down_e( bf16(silu(gate_e(x_t)) * up_e(x_t)) ),
 *   e = topk_idx[t, j].
 * x: [T, H] bf16; topk_idx/topk_scores as produced by nq_moe_route;
 * gate/up: w [E, I, H*bits/32], s/b [E, I, H/gs];
 * down:    w [E, H, I*bits/32], s/b [E, H, I/gs];  y: [T, H] bf16.
 * workspace: device buffer of nq_moe_workspace_size() bytes (caller-owned). */
int nq_moe_switch(const uint16_t *x, int64_t T, int64_t H, int64_t I,
                  int64_t E, int64_t top_k, const int32_t *topk_idx,
                  const float *topk_scores, const uint32_t *gate_w,
                  const uint16_t *gate_s, const uint16_t *gate_b,
                  const uint32_t *up_w, const uint16_t *up_s,
                  const uint16_t *up_b, const uint32_t *down_w,
                  const uint16_t *down_s, const uint16_t *down_b, int bits,
                  int group_size, void *workspace, size_t workspace_bytes,
                  uint16_t *y, void *stream);

/* Output fan-out of a tensor-parallel quantized matmul: the call computes
 * this rank's column shard and writes it into every rank's y through peer
 * pointers (CUDA IPC mappings), instead of leaving an all-gather to a
 * collective library.  No counterpart in the reference (one device); it is
 * the compute step of nq_tp_quantized_matmul_fused (nq_dist.h), which sets
 * these fields up and signals completion after it.  All pointers are valid in
 * this process (peer mappings for other ranks).  *epoch is the call number
 * (equal on every rank, increasing; read from device memory when the kernel
 * runs, so a captured CUDA graph stays correct when replayed); ready[q] ==
 * *epoch is set by rank q before its call (its earlier stream work has
 * completed), and the kernel waits for every ready flag (bounded, 2 s; a
 * timeout raises the device error word) before its first store.  The stores
 * are complete when the kernel is. */
#define NQ_MAX_RANKS 8
typedef struct nq_push {
    int nranks;
    int rank;
    const unsigned int *epoch;
    void *dst[NQ_MAX_RANKS];
    const unsigned int *ready;
} nq_push_t;

/* y_q[m, col0 + n] = (x . W^T)[m, n] on every rank q, y rows N_total apart
 * (W: this rank's N rows).  M <= 32 needs K % 256 == 0 (and not 8-bit with
 * group size 128); larger M takes the tensor-core path. */
int nq_quantized_matmul_push(const uint16_t *x, int64_t M, const uint32_t *wq,
                             const uint16_t *scales, const uint16_t *biases,
                             int64_t N, int64_t K, int bits, int group_size,
                             int64_t N_total, int64_t col0,
                             const nq_push_t *push, void *stream);

/* Every check nq_quantized_matmul_push makes before it launches (arguments,
 * alignment -- scales and biases included -- and whether a kernel serves the
 * shape with the fan-out), without launching anything: NQ_SUCCESS when the
 * call would be accepted, else the status and message it would fail with.
 * nq_tp_quantized_matmul_fused runs it before its ready kernel, so a rejected
 * call leaves the communicator's call count unchanged.  No counterpart in the
 * reference (part of the fused tensor-parallel plumbing). */
int nq_quantized_matmul_push_check(const uint16_t *x, int64_t M, const uint32_t *wq,
                                   const uint16_t *scales, const uint16_t *biases,
                                   int64_t N, int64_t K, int bits, int group_size,
                                   int64_t N_total, int64_t col0, const nq_push_t *push);

/* The switch step restricted to one shard of the experts, for expert
 * parallelism: the weights passed hold experts [e0, e0 + ne) of the E the
 * router chose from (gate/up w [ne, I, H*bits/32], down w [ne, H, ...]), and
 * the call writes, in fp32,
 *   y_partial[t] = sum over the slots j with e0 <= topk_idx[t,j] < e0 + ne of
 *                  bf16(score[t,j]) * down_e( bf16(silu(gate_e(x_t)) * up_e(x_t)) ).
 * Summing y_partial over all shards and rounding to bf16 gives nq_moe_switch's
 * result up to the order of the fp32 additions.  No counterpart in the
 * reference (which runs one device); it shards the switch step
 * compute/src/compute/model/qwen3_transformer_moe_model_mlx.cpp:29-79.
 * workspace: nq_moe_partial_workspace_size(T, E, ne, top_k, H, I) bytes. */
size_t nq_moe_partial_workspace_size(int64_t T, int64_t E, int64_t ne,
                                     int64_t top_k, int64_t H, int64_t I);
int nq_moe_switch_partial(const uint16_t *x, int64_t T, int64_t H, int64_t I,
                          int64_t E, int64_t top_k, const int32_t *topk_idx,
                          const float *topk_scores, int64_t e0, int64_t ne,
                          const uint32_t *gate_w, const uint16_t *gate_s,
                          const uint16_t *gate_b, const uint32_t *up_w,
                          const uint16_t *up_s, const uint16_t *up_b,
                          const uint32_t *down_w, const uint16_t *down_s,
                          const uint16_t *down_b, int bits, int group_size,
                          void *workspace, size_t workspace_bytes,
                          float *y_partial, void *stream);

/* Where nq_moe_switch_partial_push writes its fp32 partial sums: the call's
 * T tokens are nranks regions of rows_per_rank rows (T = nranks *
 * rows_per_rank); token q * rows_per_rank + i goes to row dst_row0 + i of
 * dst[q] (fp32, H per row; a peer mapping for another rank), and rows i >=
 * count[q] (device memory, read when the kernel runs) are padding and are not
 * written.  No counterpart in the reference: the combine step of the
 * expert-parallel switch (nq_ep_moe_switch_fused, nq_dist.h). */
typedef struct nq_rows_push {
    int nranks;
    int64_t rows_per_rank;
    int64_t dst_row0;
    const int32_t *count;
    float *dst[NQ_MAX_RANKS];
} nq_rows_push_t;

/* nq_moe_switch_partial with the partial sums written through `push`
 * instead of y_partial (same workspace size). */
int nq_moe_switch_partial_push(const uint16_t *x, int64_t T, int64_t H, int64_t I,
                               int64_t E, int64_t top_k, const int32_t *topk_idx,
                               const float *topk_scores, int64_t e0, int64_t ne,
                               const uint32_t *gate_w, const uint16_t *gate_s,
                               const uint16_t *gate_b, const uint32_t *up_w,
                               const uint16_t *up_s, const uint16_t *up_b,
                               const uint32_t *down_w, const uint16_t *down_s,
                               const uint16_t *down_b, int bits, int group_size,
                               void *workspace, size_t workspace_bytes,
                               const nq_rows_push_t *push, void *stream);

/* ---- Llama decode step ----
 * A Llama decode step on the GPU around the quantized matmuls, restating the
 * reference's compiled decode function
 * (compute/src/compute/model/llama_model.cpp:355-509): embedding row,
 * per layer RMSNorm -> q/k/v -> RoPE -> GQA attention over the growing KV
 * cache -> o (+ residual) -> RMSNorm -> gate/up -> SwiGLU -> down
 * (+ residual), final RMSNorm, LM head (lm_head, else the tied quantized
 * embedding) and a greedy argmax, whose token feeds the next step from
 * device memory as in mlx_generate_pipelined (:713-812).  Every call only
 * enqueues work on `stream` (no host synchronisation, no allocation): steps
 * may be captured in a CUDA graph and replayed.  Serves 4-bit codes with
 * hidden, intermediate and n_heads*head_dim multiples of 128, head_dim <= 256
 * and at most 8 query heads per KV head.  Weights are borrowed (they must
 * outlive the decoder) except q/k/v and gate/up, which are copied into
 * row-concatenated buffers at creation. */
typedef struct nq_qweight {
    const uint32_t *w;        /* packed codes [N, K*bits/32] (dense bf16 [N, K] for an
                                 unquantized embedding, with scales == NULL) */
    const uint16_t *scales;   /* bf16 [N, K/gs] */
    const uint16_t *biases;   /* bf16 [N, K/gs] */
} nq_qweight_t;

typedef struct nq_llama_config {
    int n_layers, hidden, n_heads, n_kv_heads, head_dim, intermediate, vocab;
    int bits, group_size, max_context;
    float rms_eps, rope_theta;
} nq_llama_config_t;

typedef struct nq_llama_layer {
    const uint16_t *input_norm;  /* bf16 [hidden], 16-byte aligned */
    const uint16_t *post_norm;   /* bf16 [hidden], 16-byte aligned */
    nq_qweight_t q, k, v, o, gate, up, down;
} nq_llama_layer_t;

typedef struct nq_llama_s *nq_llama_t;

/* lm_head NULL (or lm_head->w NULL): the tied embedding is the LM head. */
int nq_llama_create(nq_llama_t *out, const nq_llama_config_t *cfg,
                    const nq_llama_layer_t *layers, const uint16_t *final_norm,
                    const nq_qweight_t *embed, const nq_qweight_t *lm_head);
int nq_llama_destroy(nq_llama_t dec);
/* Steps enqueued since the last reset (the next step's position). */
int64_t nq_llama_position(nq_llama_t dec);
/* Empties the KV cache (position 0). */
int nq_llama_reset(nq_llama_t dec, void *stream);
/* One step on token[0] (device int32; NULL: the previous step's argmax).
 * logits (fp32 [vocab], optional) and next_token (int32, optional) receive
 * the step's logits and argmax. */
int nq_llama_step(nq_llama_t dec, const int32_t *token, float *logits,
                  int32_t *next_token, void *stream);
/* n steps over the prompt tokens[0..n) (device), or steps of a chunk each
 * after nq_llama_set_prefill_chunk; logits (optional) gets the last position's.
 * Afterwards the decoder's next input is the argmax of the last position (the
 * first generated token). */
int nq_llama_prefill(nq_llama_t dec, const int32_t *tokens, int64_t n,
                     float *logits, void *stream);
/* n greedy steps, each fed the previous step's argmax (the first one token[0]
 * when token != NULL); tokens[i] (device int32 [n]) receives step i's argmax. */
int nq_llama_generate(nq_llama_t dec, const int32_t *token, int64_t n,
                      int32_t *tokens, void *stream);

/* ---- Paged key/value cache ----
 * One layer's keys (and values): [n_pages][n_kv_heads][page_size][head_dim],
 * pages page_stride elements apart.  A contiguous cache is one page per
 * sequence.  head_dim 64, 128 or 256; page_size a multiple of 16; dtype
 * NQ_DTYPE_BF16 or NQ_DTYPE_F16; 16-byte aligned, page_stride a multiple of 8.
 *
 * The page table (device int32 [n_rows][table_ld], table_width entries used)
 * lists each sequence's pages, kv_lens [n_rows] the sequences' lengths with
 * the new tokens included.  A batch names its sequences by table row: entry b
 * is row seqs[b] (a negative one is padding), or row b when seqs is NULL.  The
 * new tokens of entry b are rows q_starts[b] .. q_starts[b + 1] of q, k, v and
 * out (device int32 [n_seqs + 1]), or row b alone when q_starts is NULL; token
 * t of n stands at position kv_lens - n + t.  Rows behind the last entry, and
 * those of padding, are neither read nor written.
 *
 * The arrays are read when the kernels run; what they say out of range (a
 * length past the table, a table row, a missing page) is cut off or read as
 * zeros and raises bit 1 of the device error word. */
typedef struct nq_paged_cache {
    void *k, *v;
    int64_t n_pages, page_stride;
    int n_kv_heads, page_size, head_dim, dtype;
} nq_paged_cache_t;

typedef struct nq_paged_batch {
    const int32_t *table;
    int64_t table_ld, table_width, n_rows;
    const int32_t *kv_lens;
    const int32_t *seqs;
    const int32_t *q_starts;
    int64_t n_seqs, n_tokens;
} nq_paged_batch_t;

/* Attention of the batch's new tokens over the cache (the keys of the new
 * tokens have been appended):
 *   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,
 *   p_j = exp(scale * q[t, h] . k[j, h / G]),  G = n_heads / n_kv_heads,
 * over the keys j <= pos(t), and j > pos(t) - window when window > 0.  A row
 * without any key (more new tokens than the length) is zero.  q and out rows:
 * [n_heads][head_dim], q_ld / out_ld elements apart (multiples of 8, 16-byte
 * aligned).  Keys and values past a sequence's length, and pages that no new
 * token's window reaches, may hold anything; the values that the rows of one
 * call see have to be finite.  A NaN in a query, or in a key that it sees, makes
 * its row NaN.  max_q: no entry has more new tokens than this (it
 * selects the kernel and the workspace's size, results hold for any; 0:
 * unknown, with the workspace that any would need).  Softmax and sums in fp32;
 * for the second product the weights are two terms of the cache's type where
 * max_q * G <= 16, and rounded to one where it is more; the result is rounded
 * once.  workspace: nq_paged_attention_workspace_size() bytes for this max_q (or
 * a larger one) and max_keys = table_width * page_size (0: none is needed),
 * 256-byte aligned, contents irrelevant; two calls that overlap on the GPU need
 * one each. */
size_t nq_paged_attention_workspace_size(int n_heads, int n_kv_heads, int head_dim, int64_t max_q,
                                         int64_t max_keys);
int nq_paged_attention(const uint16_t *q, int64_t q_ld, int n_heads, const nq_paged_cache_t *cache,
                       const nq_paged_batch_t *batch, int64_t max_q, float scale, int64_t window,
                       void *workspace, size_t workspace_bytes, uint16_t *out, int64_t out_ld,
                       void *stream);

/* Rotary positions for the new tokens' queries and keys, and their keys and
 * values into the cache.  For i < n_freqs the pair (x_i, x_{i + n_freqs}) of
 * each head of q and k is turned by pos * freqs[i] (device fp32, radians per
 * position; MLX fast::rope, traditional = false, compute/src/compute/model/
 * llama_model.cpp:446-470), the angle in 64 bits, the turn in fp32, rounded
 * once; dims past 2 * n_freqs stay.  n_freqs is a multiple of 8, at most
 * head_dim / 2; 0 turns nothing.  The queries go to q_out (may be q itself).
 * A token at a negative position or whose page is missing is not stored (error
 * word), and an entry whose row, length or starts are out of range is left out
 * (error word): it stores nothing, and its queries are not written.  Two entries of one call must not be the same sequence, nor hold their
 * new tokens' pages in common (nq_pages_reserve parts such pages): which of their
 * keys stay is not defined. */
int nq_paged_append(const uint16_t *q, int64_t q_ld, const uint16_t *k, int64_t k_ld,
                    const uint16_t *v, int64_t v_ld, int n_heads, const nq_paged_cache_t *cache,
                    const nq_paged_batch_t *batch, const float *freqs, int n_freqs, uint16_t *q_out,
                    int64_t q_out_ld, void *stream);

/* The page pool's bookkeeping, all of it in device memory, so that the calls
 * below only enqueue work (and may be captured): refs[p] sequences hold page
 * p (0: free), table and lens as above, -1 in unused table entries.  A pool is
 * [outer][n_pages][page_bytes] (outer: layers x keys and values).  Sequence
 * lists are device int32; negative entries are padding.  A list has at most
 * 2^20 entries, nq_pages_reserve's 2^16 (entries are compared with one another).
 * A refused request raises bit 2 of the device error word. */
typedef struct nq_page_table {
    int32_t *refs;
    int32_t *table;
    int32_t *lens;
    int64_t n_pages, n_rows, table_ld, table_width;
    int page_size;
} nq_page_table_t;

typedef struct nq_page_pool {
    void *data;
    int64_t outer, n_pages, page_bytes;
} nq_page_pool_t;

/* The listed sequences give their pages back and have length 0. */
int nq_pages_free(const nq_page_table_t *table, const int32_t *seqs, int64_t n, void *stream);

/* children[i] becomes a copy of parents[i] that shares all its pages.  A child
 * that has pages, is listed twice or is also a parent of this call is refused
 * (that pair alone). */
int nq_pages_fork(const nq_page_table_t *table, const int32_t *parents, const int32_t *children,
                  int64_t n, void *stream);

/* Sequence seqs[i] grows to new_lens[i] tokens: a last page that is not full
 * and has other holders is replaced by a copy, and free pages are added, the
 * lowest first, in the list's order.  All or nothing: too few free pages, a
 * length below the present one or past the table, a row out of range or a
 * sequence listed twice refuse the whole call, and lens stays as it was: an
 * append that follows has to leave these sequences out (as padding), or it writes
 * over their last tokens.  n * table_width < 2^31.
 * workspace: nq_pages_workspace_size(0, n) bytes, 256-byte aligned. */
size_t nq_pages_workspace_size(int64_t n_pages, int64_t n);
int nq_pages_reserve(const nq_page_table_t *table, const nq_page_pool_t *pool, const int32_t *seqs,
                     const int32_t *new_lens, int64_t n, void *workspace, size_t workspace_bytes,
                     void *stream);

/* The used pages past the number of used ones move into the free pages below
 * it (the k-th lowest into the k-th lowest), contents, refs and table entries:
 * the pool's upper end is free afterwards.  workspace:
 * nq_pages_workspace_size(n_pages, 0) bytes, 256-byte aligned. */
int nq_pages_compact(const nq_page_table_t *table, const nq_page_pool_t *pool, void *workspace,
                     size_t workspace_bytes, void *stream);

/* Copies pages src[i] to dst[i] in every outer slice; refs and tables are the
 * caller's.  A move whose target is also a source or an earlier target is
 * refused (that move alone). */
int nq_pages_copy(const nq_page_pool_t *pool, const int32_t *src, const int32_t *dst, int64_t n,
                  void *stream);

/* ---- Llama over a paged cache ----
 * Prompts in chunks: nq_llama_prefill passes up to `chunk` tokens through the
 * layers at a time (M-row quantized matmuls, nq_paged_attention over the
 * decoder's cache) instead of one (0, the default).  The results differ from the
 * one-token steps' by the order of the sums and the rounding of the angles, which
 * chunks take in 64 bits; from the first call with chunk > 0 on, the decoder's
 * one-token steps do so too (those captured in a graph before keep 32 bits), so
 * that queries and keys of far positions agree.  It is therefore called before a
 * sequence's first token.  Allocates the chunk's workspace; not to be called while
 * calls on the decoder are under way. */
int nq_llama_set_prefill_chunk(nq_llama_t dec, int64_t chunk);

/* The batch's new tokens (tokens: device int32 [batch->n_tokens]) through the
 * decoder's layers over a paged cache of the caller's (bf16; `cache` describes
 * layer 0, layer l's keys and values lie l * layer_stride elements on); the
 * decoder's own cache and position are not touched.  Row rows[i] of the batch
 * (device int32 [n_out]; negative: left out, its outputs are not meaningful)
 * yields logits [n_out][vocab] (fp32, optional) and next_tokens [n_out] (int32
 * argmax, optional).  Every row's token is looked up, those of padding too: one
 * outside of the vocabulary counts as 0 and raises bit 1 of the error word.
 * max_q as in nq_paged_attention.  The pages for the new
 * tokens are the caller's to reserve.  workspace: nq_llama_forward_workspace_
 * size() bytes (max_keys = table_width * page_size), 256-byte aligned. */
size_t nq_llama_forward_workspace_size(nq_llama_t dec, int64_t n_tokens, int64_t n_out, int64_t max_q,
                                       int64_t max_keys);
int nq_llama_forward(nq_llama_t dec, const int32_t *tokens, const nq_paged_cache_t *cache,
                     int64_t layer_stride, const nq_paged_batch_t *batch, int64_t max_q,
                     const int32_t *rows, int64_t n_out, float *logits, int32_t *next_tokens,
                     void *workspace, size_t workspace_bytes, void *stream);

/* nq_moe_switch without a workspace argument, for callers that cannot
 * allocate device memory themselves (an FFI host or a runtime that only
 * hands over the tensors it owns and exposes no allocator).  No counterpart
 * in the reference: it exists for those callers only.
 * Same arguments and result as nq_moe_switch; the scratch comes from a
 * static 4 MiB block inside the library (4,194,304 bytes; every GPU that
 * loads the library keeps that block until the process exits), so calls
 * whose nq_moe_workspace_size() exceeds it fail with NQ_INVALID_INPUT (at
 * the Qwen3-30B-A3B layer dims that allows up to ~50 tokens per call).  The
 * call allocates nothing.  The first call on a device looks up the block's
 * address (cudaGetSymbolAddress); make that first call before any stream
 * capture.  All calls on a device share the one block and it keeps the last
 * call's contents (the parts that must start at zero are cleared by each
 * call): calls that overlap on the GPU -- on different streams, or from
 * different threads -- race on it, so serialise them. */
int nq_moe_switch_static(const uint16_t *x, int64_t T, int64_t H, int64_t I,
                         int64_t E, int64_t top_k, const int32_t *topk_idx,
                         const float *topk_scores, const uint32_t *gate_w,
                         const uint16_t *gate_s, const uint16_t *gate_b,
                         const uint32_t *up_w, const uint16_t *up_s,
                         const uint16_t *up_b, const uint32_t *down_w,
                         const uint16_t *down_s, const uint16_t *down_b,
                         int bits, int group_size, uint16_t *y, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NQ_H_ */
