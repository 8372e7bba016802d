/*
 * lmoe_b200.h -- C ABI of the B200 (sm_100a) MoE-layer hot path.
 *
 * Plain pointers, sizes and a CUDA stream; no framework types.  Every entry point:
 *   - launches asynchronously on `stream` (never on the legacy default stream unless the
 *     caller passes it) and performs no host<->device synchronisation (except the
 *     peer-exchange setup and teardown, lmoe_p2p_alloc / _free);
 *   - never allocates device memory: outputs and workspaces are caller-owned (the one
 *     exception is the peer-exchange setup, lmoe_p2p_alloc / _open, run once per layer);
 *   - returns LMOE_OK (0), a negative LMOE_ERR_* for rejected arguments, or a positive
 *     cudaError_t value when a CUDA call failed.
 * Kernels that wait on their own pipelines bound every wait; a wait that gives up writes a
 * nonzero word into the workspace's error slot (read it with lmoe_read_error).
 *
 * Each declaration names the light-moe interface it replaces (file:line in the reference
 * repository Whitehall945/light-moe).
 */
#ifndef LMOE_B200_H_
#define LMOE_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LMOE_OK 0
#define LMOE_ERR_INVALID_ARG (-1)    /* shape / dtype / alignment / null pointer          */
#define LMOE_ERR_UNSUPPORTED (-2)    /* valid request outside what the kernels implement  */
#define LMOE_ERR_WORKSPACE (-3)      /* workspace missing or too small                    */
#define LMOE_ERR_DEVICE (-4)         /* current device is not sm_100 / kernel error word  */

/* Element types of floating-point operands (the *_typed entry points). */
#define LMOE_DTYPE_BF16 0
#define LMOE_DTYPE_F16 1
#define LMOE_DTYPE_F32 2

/* Microscaled 4-bit formats (E2M1 values with one scale byte per block of columns). */
#define LMOE_FP4_MX 0   /* blocks of 32, E8M0 (power-of-two) scales                  */
#define LMOE_FP4_NV 1   /* blocks of 16, E4M3 scales under an fp32 tensor scale      */

typedef struct CUstream_st* lmoe_stream_t; /* identical to cudaStream_t */

/* Library version as 10000*major + 100*minor + patch. */
int lmoe_version(void);

/* Human-readable text for a status code (static storage). */
const char* lmoe_status_string(int status);

/* Copies the 32-bit device error word of a router / GEMM workspace to *out (synchronises
 * `stream`).  0 means no kernel reported a problem. */
int lmoe_read_error(const void* workspace, uint32_t* out, lmoe_stream_t stream);

/* Caps the number of CTAs (one per SM) of the persistent grouped GEMMs and of the few-token layer's
 * kernels (whole pairs: two at least) launched afterwards by this process (0 = no cap: one per SM).  Leaving SMs free lets kernels on other streams
 * -- NCCL's all-to-all of the next micro-batch -- run beside a GEMM instead of after it.
 * Process-wide; read at each launch.  New (the reference has no persistent kernels). */
int lmoe_set_gemm_sm_limit(int max_ctas);
int lmoe_get_gemm_sm_limit(void);

/* ------------------------------------------------------------------------------------ */
/* Router: gate logits + fp32 softmax + top-k + renormalise + histogram / offsets /       */
/* stable permutation, in one kernel.                                                     */
/* Replaces fused_gate_topk_cuda (csrc/fused_moe_ops.cu:145-200) and the count / offset / */
/* argsort part of fused_gate_topk_permute_cuda (csrc/fused_moe_ops.cu:205-225).          */
/* ------------------------------------------------------------------------------------ */

/* Workspace bytes needed by lmoe_fused_gate_topk for these sizes. */
size_t lmoe_router_workspace_bytes(int64_t num_tokens, int num_experts);

/*
 * hidden      bf16 [num_tokens, hidden]   row-major, 16-byte aligned, hidden % 64 == 0
 * gate_weight bf16 [num_experts, hidden]  (nn.Linear layout, as the reference binding reads
 *                                          E = gate_weight.size(0), fused_moe_ops.cu:155)
 * gate_bias   fp32 [num_experts] or NULL (MoEGate(bias=True), moe_gate.py:159,171)
 * 1 <= num_experts <= 256, 1 <= top_k <= min(16, num_experts)
 * Outputs (any of the optional ones may be NULL):
 *   ids          int32 [num_tokens, top_k]  descending probability, ties -> lower id
 *   weights      fp32  [num_tokens, top_k]  renormalised to sum 1          (optional)
 *   weights_bf16 bf16  [num_tokens, top_k]  same values rounded to bf16     (optional)
 *   counts       int32 [num_experts]                                      (optional*)
 *   offsets      int32 [num_experts + 1]  exclusive scan of counts        (optional*)
 *   sorted_idx   int32 [num_tokens*top_k]  flat index t*top_k+j ordered by
 *                (expert, token, slot)                                    (optional*)
 *   positions    int32 [num_tokens*top_k]  inverse of sorted_idx: the sorted row of
 *                each flat index (optional; needs the three outputs above)
 *   logits       fp32  [num_tokens, num_experts]  gate logits (+bias), for checking
 * (*) counts, offsets and sorted_idx are produced together: pass all three or none.
 */
int lmoe_fused_gate_topk(const void* hidden, const void* gate_weight, const float* gate_bias,
                         int64_t num_tokens, int hidden_size, int num_experts, int top_k,
                         int32_t* ids, float* weights, void* weights_bf16,
                         int32_t* counts, int32_t* offsets, int32_t* sorted_idx,
                         int32_t* positions, float* logits,
                         void* workspace, size_t workspace_bytes, lmoe_stream_t stream);

/* lmoe_fused_gate_topk for hidden states and gate weight of any of the LMOE_DTYPE_* types
 * (x_dtype, w_dtype), as the reference's binding accepts any floating dtype and computes the
 * logits in fp32 from the converted operands (csrc/fused_moe_ops.cu:158-159):
 *   - both bf16 or both fp16: tensor-core logits (16-bit products are exact in fp32, fp32
 *     accumulation);
 *   - otherwise (fp32 on either side, or bf16 with fp16): fp32 logits on CUDA cores from the
 *     caller's values, each a sequential fp32 sum over the hidden dimension.
 * probs (optional, fp32 [num_tokens, num_experts]) receives the full softmax probabilities,
 * the router_probs of the reference's RoutingOutput (python/light_moe/ops/moe_gate.py:20-36)
 * used by its load-balancing loss (:80-122); bit-identical to the values the top-k selects
 * from.  Workspace: lmoe_router_workspace_bytes_typed().  Everything else as
 * lmoe_fused_gate_topk. */
size_t lmoe_router_workspace_bytes_typed(int64_t num_tokens, int num_experts, int x_dtype, int w_dtype);

int lmoe_fused_gate_topk_typed(const void* hidden, int x_dtype, const void* gate_weight, int w_dtype,
                               const float* gate_bias, int64_t num_tokens, int hidden_size, int num_experts,
                               int top_k, int32_t* ids, float* weights, void* weights_bf16,
                               int32_t* counts, int32_t* offsets, int32_t* sorted_idx,
                               int32_t* positions, float* logits, float* probs,
                               void* workspace, size_t workspace_bytes, lmoe_stream_t stream);

/* lmoe_fused_gate_topk without a workspace argument (no counterpart in the reference): the
 * scratch lives in a fixed 1.25 MB device array inside this library, for callers that may
 * not allocate device memory (an allocator that owns all device memory, a serving loop that
 * forbids allocation after start-up).
 *   - num_tokens <= 16384 (any num_experts <= 256); larger calls return LMOE_ERR_WORKSPACE.
 *   - The first call on a device looks up the array's device address; make that first call
 *     before any stream capture.  Later calls allocate nothing.
 *   - All calls on a device share the one array, which keeps whatever the last call left in
 *     it (each call clears the parts that must start at zero).  Calls that overlap in time,
 *     on different streams or host threads, race on it: serialise them.
 *   - A wait timeout recorded by the kernel stays in the shared array; use
 *     lmoe_fused_gate_topk with a workspace when the device error word must be read.
 * Other arguments, outputs and status codes as lmoe_fused_gate_topk. */
int lmoe_fused_gate_topk_static(const void* hidden, const void* gate_weight, const float* gate_bias,
                                int64_t num_tokens, int hidden_size, int num_experts, int top_k,
                                int32_t* ids, float* weights, void* weights_bf16,
                                int32_t* counts, int32_t* offsets, int32_t* sorted_idx,
                                int32_t* positions, float* logits, lmoe_stream_t stream);

/* ------------------------------------------------------------------------------------ */
/* Row gather / weighted combine                                                          */
/* ------------------------------------------------------------------------------------ */

/* permuted[r, :] = hidden[sorted_idx[r] / top_k, :] for r < rows; elements of elem_bytes
 * (2 or 4) bytes, hidden_size * elem_bytes a multiple of 16, rows copied unchanged.
 * Replaces the expand + index_select of fused_gate_topk_permute_cuda
 * (csrc/fused_moe_ops.cu:227-228) and permute_tokens (python/light_moe/ops/grouped_gemm.py:
 * 202-247). */
int lmoe_permute_rows(const void* hidden, int elem_bytes, const int32_t* sorted_idx, int64_t rows,
                      int hidden_size, int top_k, void* permuted, lmoe_stream_t stream);

/* ------------------------------------------------------------------------------------ */
/* int4 weight format (defined by this library; the reference only has the unused flag    */
/* EngineConfig.use_int4_quantization, python/light_moe/engine/executor.py:44-48).        */
/*   qweight uint8 [rows, K/2]: byte b holds k=2b (low nibble) and k=2b+1 (high nibble),   */
/*           each stored as q+8;  scales fp16 [rows, K/group]: s = fp16(max|w|/7);          */
/*   q = clamp(rint(w / s), -8, 7);  dequantised value = bf16_rn(q * s).                   */
/* ------------------------------------------------------------------------------------ */

/* w: [rows, K] bf16 (w_is_fp32 == 0) or fp32 (w_is_fp32 != 0). */
int lmoe_quantize_w4(const void* w, int w_is_fp32, int64_t rows, int K, int group_size,
                     uint8_t* qweight, uint16_t* scales, lmoe_stream_t stream);

/* out: bf16 [rows, K]. */
int lmoe_dequantize_w4(const uint8_t* qweight, const uint16_t* scales, int64_t rows, int K,
                       int group_size, void* out, lmoe_stream_t stream);

/* Bytes of the device ("prepacked") layout streamed by the W4A16 GEMM for `num_experts`
 * matrices of [rows, K]: super-blocks of 128 rows x 128 K values with their fp16 scales
 * embedded, expert-major.  paired != 0 interleaves two such matrices (gate w1 and up w3) by
 * 64-row blocks, giving 2*rows rows.  K % 128 == 0; group_size a multiple of 64 that
 * divides 128 or is a multiple of it; rows % 128 == 0 (rows % 64 == 0 when paired). */
int lmoe_w4_prepacked_bytes(int num_experts, int rows, int K, int group_size, int paired,
                            size_t* packed_bytes);

/* Canonical int4 weights [num_experts, rows, K/2] + scales -> prepacked layout.  Pass the
 * up-projection as qweight_b / scales_b to build the paired gate/up layout, else NULL. */
int lmoe_prepack_w4(const uint8_t* qweight_a, const uint16_t* scales_a,
                    const uint8_t* qweight_b, const uint16_t* scales_b,
                    int num_experts, int rows, int K, int group_size,
                    uint8_t* packed, lmoe_stream_t stream);

/* ------------------------------------------------------------------------------------ */
/* Grouped GEMMs.  Rows [offsets[e], offsets[e+1]) of `input` (bf16 [total_rows, K]) are  */
/* multiplied by expert e's weight matrix ([N, K]); offsets are int32 or int64 [E+1] and  */
/* are read on the device (no host copy).  Workspace: lmoe_gemm_workspace_bytes().        */
/* ------------------------------------------------------------------------------------ */

size_t lmoe_gemm_workspace_bytes(void);

/* Dense weights [num_experts, N, K] of the input's type.  output [total_rows, N] of the
 * same type; with zero_fill the rows outside every expert range are zeroed first.
 * dtype LMOE_DTYPE_BF16 / LMOE_DTYPE_F16: tcgen05 tensor cores (exact 16-bit products, fp32
 * accumulation, K % 64 == 0); LMOE_DTYPE_F32: fp32 FFMA on CUDA cores (K % 4 == 0), as the
 * reference's fp32 cuBLAS GEMM computes in fp32.
 * Replaces grouped_gemm_cuda (csrc/grouped_gemm.cu:11-43), which zero-fills (:24), copies
 * the offsets to the host (:27) and runs one cuBLAS GEMM per expert in the input dtype
 * (:30-40). */
int lmoe_grouped_gemm(const void* input, int dtype, int64_t total_rows, int K, const void* weights, int N,
                      const void* expert_offsets, int offsets_are_int64, int num_experts,
                      int zero_fill, void* output, void* workspace, size_t workspace_bytes,
                      lmoe_stream_t stream);

/* lmoe_grouped_gemm with dtype LMOE_DTYPE_BF16. */
int lmoe_grouped_gemm_bf16(const void* input, int64_t total_rows, int K, const void* weights, int N,
                           const void* expert_offsets, int offsets_are_int64, int num_experts,
                           int zero_fill, void* output, void* workspace, size_t workspace_bytes,
                           lmoe_stream_t stream);

/* W4A16: prepacked int4 weights (N rows per expert, N % 128 == 0, K % 128 == 0), fp32
 * accumulation.
 * epilogue 0: output[r, n] = acc                               (ldo >= N)
 * epilogue 1: SwiGLU over a paired gate/up matrix of N = 2*F rows:
 *             output[r, f] = silu(gate[r, f]) * up[r, f]         (ldo >= F)
 * epilogue 2: output[dest_rows[r], n] = row_scale[r] * acc       (NULL = identity / 1)
 * segment_expert: weight matrix used by each of the num_experts row segments (NULL: the
 *             identity), so rows grouped by (source, expert) need no re-sort; -1 marks a
 *             hole (padding rows of a fixed-capacity exchange): its rows are skipped and
 *             their output rows are left untouched.
 * num_weight_matrices: matrices held by `packed`; every segment_expert entry (or, without a
 *             map, every segment index) must lie in [0, num_weight_matrices).  A kernel that
 *             finds an entry outside it, or offsets that decrease or pass total_rows, skips
 *             that segment and writes a nonzero error word into the workspace
 *             (lmoe_read_error).
 * max_rows_per_expert: an upper bound of any expert's row count if known (0 = unknown);
 * small bounds select the decode-sized tiles.
 * New op; the reference has no W4A16 GEMM (SparseMoEBlockFast's GroupedLinear calls,
 * python/light_moe/model/moe_block.py:249-256, are its dense counterpart). */
int lmoe_w4a16_grouped_gemm(const void* input, int64_t total_rows, int K, const uint8_t* packed,
                            int N, int group_size,
                            const void* expert_offsets, int offsets_are_int64, int num_experts,
                            const int32_t* segment_expert, int num_weight_matrices,
                            int epilogue, const int32_t* dest_rows, const float* row_scale,
                            int64_t max_rows_per_expert, void* output, int64_t ldo,
                            void* workspace, size_t workspace_bytes, lmoe_stream_t stream);

/* Gradients of lmoe_grouped_gemm, y[r, n] = sum_k input[r, k] * weights[e, n, k], for the rows
 * [offsets[e], offsets[e + 1]) of expert e; dtype of all operands LMOE_DTYPE_* (bf16 and fp16 on
 * tensor cores with fp32 accumulation; fp32 as sums of bf16 products of fp32 accuracy on tensor
 * cores, or in fp32 on CUDA cores); any N, K >= 1.  total_rows, N and K up to 2^31 - 1025.
 *   dgrad: grad_input [total_rows, K] = grad_output [total_rows, N] * weights [E, N, K] of the
 *          row's expert; rows outside every expert are zero
 *   wgrad: grad_weights [E, N, K] (out_dtype: dtype or LMOE_DTYPE_F32), the sum over the
 *          expert's rows of grad_output^T * input; experts without rows are zero
 * 16-bit operands with row lengths that are multiples of 8 are read where they lie and must be
 * 16-byte aligned; other row lengths are copied into the workspace first.  fp32 activations are
 * written to the workspace as three bf16 planes each, unless the product is small; without a
 * workspace (NULL) fp32 operands take the CUDA cores.  Few rows with a long contraction are summed
 * in ranges, whose sums lie in the workspace too; where only the copies fit, in one.
 * lmoe_grouped_gemm_grad_workspace_bytes: 0 where none is needed.  Operands that are not finite give
 * results that are not finite (fp32 on tensor cores: NaN where fp32 may give an infinity).  The tensor
 * cores' fp32 sums of 16-bit products truncate where they add: sums of one sign come out low by up to
 * 2^-23 a product (measured: 2.5e-5 of 8192 products, 3.4e-4 of 65536).  The lowest of the three planes ends at 2^-133, so fp32 operands
 * below 2^-107 count with an error of up to 2^-134 each on tensor cores.
 * error: a device word that the caller has zeroed, or NULL.  Offsets that decrease or leave
 * [0, total_rows] set it, and every row then counts as outside every expert.
 * The reference's backward is autograd through one mm_out per expert (csrc/grouped_gemm.cu:30-40,
 * python/light_moe/ops/grouped_gemm.py:65-106). */
/* form: 0 dgrad, 1 wgrad, 2 lmoe_grouped_gemm_any. */
size_t lmoe_grouped_gemm_grad_workspace_bytes(int form, int dtype, int64_t total_rows, int N, int K, int num_experts);
int lmoe_grouped_gemm_dgrad(const void* grad_output, int dtype, int64_t total_rows, int N, const void* weights, int K,
                            const void* expert_offsets, int offsets_are_int64, int num_experts, void* grad_input,
                            void* workspace, size_t workspace_bytes, uint32_t* error, lmoe_stream_t stream);
int lmoe_grouped_gemm_wgrad(const void* grad_output, int dtype, int64_t total_rows, int N, const void* input, int K,
                            const void* expert_offsets, int offsets_are_int64, int num_experts, int out_dtype,
                            void* grad_weights, void* workspace, size_t workspace_bytes, uint32_t* error,
                            lmoe_stream_t stream);

/* lmoe_grouped_gemm for any N, K >= 1 (that entry wants K a multiple of 128, or for fp32 of 4): output
 * [total_rows, N], zero outside every expert; sizes, workspace and error as for the gradients. */
int lmoe_grouped_gemm_any(const void* input, int dtype, int64_t total_rows, int K, const void* weights, int N,
                          const void* expert_offsets, int offsets_are_int64, int num_experts, void* output,
                          void* workspace, size_t workspace_bytes, uint32_t* error, lmoe_stream_t stream);

/* ------------------------------------------------------------------------------------ */
/* Microscaled 4-bit floating point.  A row of K values (K % 32 == 0) is K/2 bytes of E2M1   */
/* codes (even column in the low nibble; code magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6, sign in  */
/* bit 3) and one scale byte per block; scale rows are lmoe_fp4_scale_pitch(K) bytes apart   */
/* (K / block padded to a multiple of 32, the padding zero).                                 */
/*   LMOE_FP4_MX: byte = clamp(floor(log2 max|x|) - 2, -127, 127) + 127, scale 2^(byte-127)   */
/*   LMOE_FP4_NV: scale s * g, s = E4M3(max|x| / (6 g)) (at most 448), g the tensor scale     */
/* code = x / scale to the nearest code, ties to even, at most 6 (0 where s is 0).            */
/* A block with an infinity or a NaN (or a g that is not positive and finite) gets the NaN   */
/* scale byte (255 / 127) and zero codes, so it reads as NaN.                                 */
/* The reference has no 4-bit floating point.                                                 */
/* ------------------------------------------------------------------------------------ */

/* Bytes between scale rows, or LMOE_ERR_INVALID_ARG. */
int lmoe_fp4_scale_pitch(int K, int format);

/* x: [rows, K] of LMOE_DTYPE_*, rows ldx elements apart.  global_scale (LMOE_FP4_NV; NULL = 1):
 * one fp32 value per rows_per_scale rows.  positions (optional): int32 [rows, copies], the output
 * rows that row r is written to (entries outside [0, out_rows) are skipped); without it copies
 * = 1 and out_rows = rows.  q [out_rows, K/2] 16-byte aligned; scales [out_rows, pitch], 2-byte aligned. */
int lmoe_quantize_fp4(const void* x, int dtype, int64_t rows, int K, int64_t ldx, int format,
                      const float* global_scale, int64_t rows_per_scale, const int32_t* positions, int copies,
                      int64_t out_rows, uint8_t* q, uint8_t* scales, lmoe_stream_t stream);

/* q and out (bf16 [rows, K]) 16-byte aligned; scale rows scale_pitch bytes apart. */
int lmoe_dequantize_fp4(const uint8_t* q, const uint8_t* scales, int64_t scale_pitch, int64_t rows, int K, int format,
                        const float* global_scale, int64_t rows_per_scale, void* out, lmoe_stream_t stream);

/* Grouped product of 4-bit operands: for the rows r of expert e
 *   output[r, n] = alpha[e] * sum_k x[r, k] * w[e, n, k]                      (wq_up == NULL)
 *   output[r, n] = silu(alpha[e] * x . w[e, n]) * (alpha_up[e] * x . up[e, n])   otherwise
 * exact products, fp32 sums that truncate where they add (2e-6 low after 14336 products of one sign under
 * nvfp4, at most 2^-23 a product).  x: codes xq [total_rows, K/2], scales xs; w (and up): codes
 * [E, N, K/2], scales [E, N, ws_pitch]; both operands of the same format, pitches multiples of 32
 * and at least lmoe_fp4_scale_pitch, codes 16-byte and scales 32-byte aligned.  alpha, alpha_up: fp32 [E] or NULL
 * (1): the product of the two tensor scales.  output [total_rows, N] of out_dtype; rows outside
 * every expert are zero.  total_rows, N and K up to 2^31 - 1025.  error: as above. */
int lmoe_fp4_grouped_gemm(const uint8_t* xq, const uint8_t* xs, int64_t xs_pitch, int64_t total_rows, int K,
                          const uint8_t* wq, const uint8_t* ws, const uint8_t* wq_up, const uint8_t* ws_up,
                          int64_t ws_pitch, int N, int format, const void* expert_offsets, int offsets_are_int64,
                          int num_experts, const float* alpha, const float* alpha_up, int out_dtype, void* output,
                          uint32_t* error, lmoe_stream_t stream);

/* ------------------------------------------------------------------------------------ */
/* 8-bit floating point (E4M3) with one fp32 scale per block of 128 columns: of one row        */
/* (activations) or of 128 rows (weights).  The last blocks may be partial; K % 16 == 0, at most 2^31 - 8208. */
/*   s = max(max|x| / 448, 2^-126), or with power_of_two the next power of two; code = x / s to */
/*   the nearest E4M3 value, ties to even; a block with an infinity or a NaN gets the scale NaN  */
/*   and zero codes, so it reads as NaN.                                                        */
/* The reference has no 8-bit floating point.                                                  */
/* ------------------------------------------------------------------------------------ */

/* Blocks of one row.  x: [rows, K] of LMOE_DTYPE_*, rows ldx elements apart.  positions (optional): int32
 * [rows, copies], the output rows that row r is written to (entries outside [0, out_rows) are skipped);
 * without it copies = 1 and out_rows = rows.  q [out_rows, K] 16-byte aligned; the scale of row r and
 * block b at scales[b * scale_pitch + r], scale_pitch >= out_rows. */
int lmoe_quantize_fp8(const void* x, int dtype, int64_t rows, int K, int64_t ldx, int power_of_two,
                      const int32_t* positions, int copies, int64_t out_rows, uint8_t* q, float* scales,
                      int64_t scale_pitch, lmoe_stream_t stream);

/* Blocks of 128 x 128 of `count` matrices [rows, K]: q [count, rows, K] 16-byte aligned, scales [count,
 * ceil(rows / 128), ceil(K / 128)]. */
int lmoe_quantize_fp8_blocks(const void* x, int dtype, int64_t count, int64_t rows, int K, int power_of_two,
                             uint8_t* q, float* scales, lmoe_stream_t stream);

/* q and out ([count, rows, K] of out_dtype) 16-byte aligned; block_rows 1 or 128; strides of the scales in
 * elements between matrices, row blocks and column blocks. */
int lmoe_dequantize_fp8(const uint8_t* q, const float* scales, int64_t scale_mat_stride, int64_t scale_row_stride,
                        int64_t scale_block_stride, int64_t count, int64_t rows, int K, int block_rows, int out_dtype,
                        void* out, lmoe_stream_t stream);

/* Grouped product of such operands: for the rows r of expert e
 *   output[r, n] = sum_b xs[b, r] * ws[e, n / 128, b] * (x . w[e, n] over block b)   (wq_up == NULL)
 *   output[r, n] = silu(x . w[e, n]) * (x . up[e, n])                                  otherwise
 * exact products, fp32 sums of a block on the tensor cores, fp32 sums over the blocks rounded to nearest.
 * x: codes xq [total_rows, K], scales xs [K blocks][xs_pitch]; w (and up): codes [E, N, K], scales
 * [E, ceil(N / 128), ceil(K / 128)]; codes 16-byte aligned.  The product of the two scales of a block has to
 * be an fp32 number too (a factor that overflows makes NaN of sums that are zero).  output [total_rows, N] of out_dtype; rows
 * outside every expert are zero.  total_rows and K up to 2^31 - 1025, N up to 2^30 - 513.  error: as above; should a
 * bounded wait ever run out, what was not computed is NaN. */
int lmoe_fp8_grouped_gemm(const uint8_t* xq, const float* xs, int64_t xs_pitch, int64_t total_rows, int K,
                          const uint8_t* wq, const float* ws, const uint8_t* wq_up, const float* ws_up, int N,
                          const void* expert_offsets, int offsets_are_int64, int num_experts, int out_dtype,
                          void* output, uint32_t* error, lmoe_stream_t stream);

/* A whole MoE layer for at most 16 tokens in two kernels: router (softmax, top-k with ties to the lower
 * id, renormalised weights), y[t] = sum_j weights[t, j] * w2 (silu(w1 x) * (w3 x)) of expert ids[t, j], plus
 * the num_shared experts behind the routed ones (weight 1).
 *   x [num_tokens, hidden_size], gate_weight [num_experts, hidden_size] of dtype (LMOE_DTYPE_BF16 or _F16),
 *     16-byte aligned; gate_bias fp32 [num_experts] or NULL
 *   w1, w3 [E + S, ffn, hidden], w2 [E + S, hidden, ffn], 32-byte aligned: of dtype, or (with the three
 *     scales) E4M3 codes with fp32 scales of blocks of 128 x 128 as lmoe_quantize_fp8_blocks writes them
 *   y [num_tokens, hidden_size] of dtype; ids int32, weights fp32 [num_tokens, top_k]
 * Hidden values stay in fp32 between the kernels and enter the second product as a sum of two fp16 numbers (22
 * bits), or with dense bf16 weights of three bf16 numbers; all sums are fp32.  Values below 2^-39 of a token's largest (bf16 tokens with E4M3 weights) or
 * of its largest hidden value over all of its experts (fp16 products) are lost, and block scales of 2^84 and more may
 * overflow the scaled sums.  Routing weights are NaN where the softmax has no value (a logit of +inf, or nothing but -inf).
 * hidden_size % 64 == 0, at most 16384; ffn_size % 32 == 0, at most 65536; num_experts <= 256, top_k <= 16,
 * num_shared <= 16; LMOE_ERR_UNSUPPORTED where eight tokens of that hidden size do not fit shared memory
 * (from about 11000 on for eight).  The result does not depend on timing; should a bounded wait of the kernels ever run
 * out, y is NaN.  The workspace
 * (lmoe_few_tokens_workspace_bytes; 0 for sizes that are refused), 16-byte aligned, need not be cleared;
 * calls that may run at the same time need one each. */
size_t lmoe_few_tokens_workspace_bytes(int64_t num_tokens, int hidden_size, int ffn_size, int num_experts, int top_k,
                                       int num_shared);
int lmoe_moe_layer_few_tokens(const void* x, int dtype, int64_t num_tokens, int hidden_size, const void* gate_weight,
                              const float* gate_bias, int num_experts, int top_k, int num_shared, const void* w1,
                              const void* w3, const void* w2, const float* w1_scales, const float* w3_scales,
                              const float* w2_scales, int ffn_size, void* y, int32_t* ids, float* weights,
                              void* workspace, size_t workspace_bytes, lmoe_stream_t stream);

/* Weighted combine of per-slot expert rows back to tokens:
 *   y[t, :] = sum_j weights[t*top_k+j] * rows[positions[t*top_k+j], :]
 *             + sum_s extra_rows[s*num_tokens + t, :]
 * fp32 accumulation in slot order, bf16 in / out, hidden_size even.
 * Replaces unpermute_tokens (python/light_moe/ops/grouped_gemm.py:250-279) and the
 * expert-parallel unsort + weighted sum (python/light_moe/distributed/expert_parallel.py:
 * 307-317). */
/* Fixed-capacity expert-parallel exchange (decode): every rank sends every rank a block of
 * capacity_rows = capacity_tokens * top_k rows, so the all-to-alls have equal splits and no
 * count reaches the host.  All arrays are device int32.
 * Send plan: counts [ep * experts_per_rank] rows of this rank per (destination rank, local
 * expert) in router order; sorted_idx / positions the router's order and its inverse
 * [num_tokens * top_k]. Writes send_index [ep * capacity_rows] (the sorted row carried by each
 * slot of each destination's block, 0 for padding: gather rows with lmoe_permute_rows) and
 * combine_pos [num_tokens * top_k] (the slot, in the returned blocks, of each (token, choice):
 * the positions argument of lmoe_combine_rows). num_tokens * top_k <= capacity_rows.
 * Receive plan: recv_counts [ep * experts_per_rank] rows received per (source rank, local
 * expert). Writes regroup [ep * capacity_rows] (received row at each expert-major position:
 * expert 0 from every source, expert 1, ..., then all padding), restore (its inverse) and
 * seg_offsets [experts_per_rank + num_shared + 2] (the local experts' segments, one padding
 * hole for segment map entry -1, then num_shared segments of num_tokens rows).
 * New: the reference pads to equal splits by sending every token to every rank
 * (python/light_moe/distributed/expert_parallel.py:186-244). */
int lmoe_capacity_send_plan(const int32_t* counts, const int32_t* sorted_idx, const int32_t* positions,
                            int64_t num_tokens, int top_k, int ep, int experts_per_rank, int64_t capacity_rows,
                            int32_t* send_index, int32_t* combine_pos, lmoe_stream_t stream);
int lmoe_capacity_receive_plan(const int32_t* recv_counts, int ep, int experts_per_rank, int64_t capacity_rows,
                               int num_shared, int64_t num_tokens, int32_t* regroup, int32_t* restore,
                               int32_t* seg_offsets, lmoe_stream_t stream);

/* Expert-parallel exchange over peer memory (NVLink), replacing the NCCL all-to-alls of    */
/* python/light_moe/distributed/expert_parallel.py:186-244 and :275-319.  Every rank         */
/* allocates one buffer of lmoe_p2p_buffer_bytes (same geometry on all ranks; Tc = the      */
/* capacity_tokens every rank passes, num_tokens <= Tc per step) with lmoe_p2p_alloc, sends  */
/* the 64-byte IPC handle to the others, maps theirs with lmoe_p2p_open and keeps a device   */
/* array peers[ep] of the mapped bases (its own allocation at peers[me]).  One step:          */
/*   lmoe_p2p_exchange_counts  counts[E] (the router's) -> seg_offsets[E/ep + 2 + S], the     */
/*                             local segments (experts, a hole, S shared segments of T rows)  */
/*                             of the rows region, and dst_base[E] (scratch for dispatch)     */
/*   lmoe_p2p_dispatch         x rows in router order straight into the owners' rows regions */
/*   lmoe_p2p_wait(which = 1)  the rows of every peer arrived: run the grouped GEMMs on the   */
/*                             rows region (at rows_offset; segment e's weight: experts        */
/*                             0..E/ep-1, -1 for the hole, then the shared experts)           */
/*   lmoe_p2p_send_back        the down GEMM's routed output rows back to their sources' ret  */
/*                             regions (slot t*k + j)                                         */
/*   lmoe_p2p_wait(which = 2)  every routed output of this rank's tokens is in its ret region */
/*                             (at ret_offset): lmoe_combine_rows with positions = slot       */
/* state: int32[4] on the device, zeroed once ([0] step epoch, [1] error word: nonzero when a  */
/* wait ran out of time or counts were inconsistent, [2], [3] internal counters).  Waits are  */
/* bounded (2 s); every rank must run every step, in the same order.  lmoe_p2p_alloc / _free */
/* / _open / _close are the library's only entry points that allocate, map or free device    */
/* memory (and synchronise the device): call them at setup and teardown, never in a step.    */
size_t lmoe_p2p_buffer_bytes(int ep, int num_experts, int64_t capacity_tokens, int top_k, int num_shared,
                             int hidden);
int lmoe_p2p_buffer_offsets(int ep, int num_experts, int64_t capacity_tokens, int top_k, int num_shared,
                            int hidden, size_t* rows_offset, size_t* ret_offset);
int lmoe_p2p_alloc(size_t bytes, void** ptr, void* ipc_handle);
int lmoe_p2p_open(const void* ipc_handle, void** ptr);
int lmoe_p2p_close(void* ptr);
int lmoe_p2p_free(void* ptr);
int lmoe_p2p_exchange_counts(const uint64_t* peers, int me, int ep, int num_experts, int64_t capacity_tokens,
                             int top_k, int num_shared, int hidden, int64_t num_tokens, int32_t* state,
                             const int32_t* counts, int32_t* seg_offsets, int32_t* dst_base,
                             lmoe_stream_t stream);
int lmoe_p2p_dispatch(const uint64_t* peers, int me, int ep, int num_experts, int64_t capacity_tokens, int top_k,
                      int num_shared, int hidden, int64_t num_tokens, int32_t* state, const void* x,
                      const int32_t* sorted_idx, const int32_t* ids, const int32_t* offsets,
                      const int32_t* dst_base, lmoe_stream_t stream);
int lmoe_p2p_wait(const uint64_t* peers, int me, int ep, int num_experts, int64_t capacity_tokens, int top_k,
                  int num_shared, int hidden, int64_t num_tokens, int32_t* state, int which, lmoe_stream_t stream);
int lmoe_p2p_send_back(const uint64_t* peers, int me, int ep, int num_experts, int64_t capacity_tokens, int top_k,
                       int num_shared, int hidden, int64_t num_tokens, int32_t* state, const void* out,
                       const int32_t* seg_offsets, lmoe_stream_t stream);

/* Setup once after mapping the peers (shared experts' destinations in this rank's buffer).  */
int lmoe_p2p_init(const uint64_t* peers, int me, int ep, int num_experts, int64_t capacity_tokens, int top_k,
                  int num_shared, int hidden, int32_t* state, lmoe_stream_t stream);
/* The down projection fused with the return transfer (prefill-sized steps, in place of      */
/* lmoe_p2p_send_back): the W4A16 grouped GEMM on h [rows region rows, ffn_size] (the gate/up */
/* output of the rows region) whose epilogue writes each routed output row straight into its  */
/* source rank's ret slot over NVLink and each shared-expert row into dest_bases[ep]          */
/* ([S * num_tokens, hidden] bf16 of this rank); dest_bases[r < ep] = peers[r] + ret_offset. */
/* Then the sources' return flags are raised.  buffer = this rank's own allocation.           */
int lmoe_p2p_down_gemm(const uint64_t* peers, int me, int ep, int num_experts, int64_t capacity_tokens, int top_k,
                       int num_shared, int hidden, int64_t num_tokens, int32_t* state, void* buffer,
                       const void* h, int ffn_size, const uint8_t* w2_packed, int group_size,
                       const int32_t* seg_offsets, const int32_t* seg_expert, int num_segments,
                       int num_weight_matrices, const uint64_t* dest_bases, lmoe_stream_t stream);

int lmoe_combine_rows(const void* rows, const int32_t* positions, const float* weights,
                      int64_t num_tokens, int top_k, int hidden_size,
                      const void* extra_rows, int num_extra, void* y, lmoe_stream_t stream);

/* ------------------------------------------------------------------------------------ */
/* The W4A16 MoE layer: router -> gather -> gate/up GEMM (SwiGLU) -> down GEMM (routing   */
/* weight, scatter to slot) -> per-token combine, all on `stream` without host syncs.     */
/* Replaces SparseMoEBlock.forward / SparseMoEBlockFast.forward                           */
/* (python/light_moe/model/moe_block.py:119-169, :216-274) with int4 experts.             */
/* ------------------------------------------------------------------------------------ */

size_t lmoe_moe_layer_workspace_bytes(int64_t num_tokens, int hidden_size, int ffn_size,
                                      int num_experts, int top_k, int num_shared);

/*
 * x        bf16 [num_tokens, hidden_size]    (hidden_size % 128 == 0, ffn_size % 128 == 0)
 * gate_*   router weight bf16 [num_experts, hidden_size], optional fp32 bias
 * w13      paired prepacked gate/up weights of num_experts + num_shared experts
 *          (routed experts first), each 2*ffn_size x hidden_size
 * w2       prepacked down weights, each hidden_size x ffn_size
 * num_shared always-on experts (weight 1, every token), 0 for Mixtral
 * y        bf16 [num_tokens, hidden_size], 8-byte aligned
 * ids_out / weights_out: optional copies of the routing (int32 / fp32 [num_tokens, top_k])
 */
int lmoe_moe_layer_w4a16(const void* x, int64_t num_tokens, int hidden_size,
                         const void* gate_weight, const float* gate_bias, int num_experts,
                         int top_k, int num_shared,
                         const uint8_t* w13_packed, const uint8_t* w2_packed,
                         int ffn_size, int group_size, void* y,
                         int32_t* ids_out, float* weights_out,
                         void* workspace, size_t workspace_bytes, lmoe_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* LMOE_B200_H_ */
