/*
 * C ABI of the f32 operators that run between the W4A32 Linears of a Qwen2-style decoder, and of a
 * decoder runner built from them (one call = prefill of a prompt, or one greedy decode step).
 * Same conventions as w4a32_hip.h: d_* pointers are device memory, calls only enqueue on
 * `stream`, nothing allocates, synchronises or exits; the return value is a W4A32_* code.
 *
 * Positions and lengths are read from device memory, so a decode step is one fixed launch
 * sequence that a caller may capture into a HIP graph and replay per token.
 */
#ifndef W4A32_DECODER_H
#define W4A32_DECODER_H

#include "w4a32_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- operators ------------------------------------------------------------------------- */

/* d_out[m][:] = d_table[d_ids[m]][:]  (f32 rows of D, int64 ids clamped to [0, vocab)).
 * LLMEmbeddingTokenOp::forward, mllm/Backends/Arm/Ops/LLMEmbeddingTokenOp.cpp:24-50. */
int w4a32_op_embedding(const int64_t* d_ids, const float* d_table, int M, int D, int vocab,
                       float* d_out, void* stream);

/* h_out = h + delta (skipped when d_delta is NULL); y = h_out * (w * 1/sqrt(mean(h_out^2) + eps)).
 * d_h_out may alias d_h. D % 4 == 0.
 * ArmRMSNormOp::forward, mllm/Backends/Arm/Ops/RMSNormOp.cpp:36-76, with the residual add of
 * QWenDecoder::forward (mllm/Models/ds_qwen2/modeling_ds_qwen2.hpp:175-183) in front. */
int w4a32_op_rmsnorm(const float* d_h, const float* d_delta, const float* d_weight, int M, int D,
                     float eps, float* d_h_out, float* d_y, void* stream);

/* out = a + b; out = silu(gate) * up (QWenMLP::forward, modeling_ds_qwen2.hpp:47-54). n % 4 == 0.
 * silu(g) * u is evaluated as g * rcp(1 + exp2(-g * log2 e)) * u with the hardware's exponential and
 * reciprocal (about 1 ulp each, 3e-7 relative against the correctly rounded expression), the same
 * expression in every kernel of this library that applies it. */
int w4a32_op_add(const float* d_a, const float* d_b, float* d_out, size_t n, void* stream);
int w4a32_op_silu_mul(const float* d_gate, const float* d_up, float* d_out, size_t n, void* stream);

/* The two operators above with the row quantiser of the Linear that reads their result behind them
 * (w4a32_quant_lhs, include/w4a32_hip.h): the f32 rows they would write are never stored, the
 * quantised rows go to d_ws for w4a32_matmul_quantized*(). For M > 8 rows of K <= 16384 values.
 *   norm:     h_out = h + delta (skipped when d_delta is NULL; d_h_out may alias d_h), then the
 *             rows h_out * (w * 1/sqrt(mean(h_out^2) + eps)) are quantised;
 *   silu_mul: the rows silu(gate) * up are quantised.
 * The reference runs RMSNormOp / the MLP's elementwise ops and the Linear's own row quantiser as
 * separate passes (RMSNormOp.cpp:36-76, modeling_ds_qwen2.hpp:47-54, kai_linear.cpp:358-362). */
int w4a32_quant_lhs_norm(const float* d_h, const float* d_delta, const float* d_weight, float eps,
                         float* d_h_out, int M, int K, void* d_ws, void* stream);
int w4a32_quant_lhs_silu_mul(const float* d_gate, const float* d_up, int M, int K, void* d_ws,
                             void* stream);

/* A Linear that runs split over K (w4a32_splitk_scratch_bytes(M, K, N) != 0, include/w4a32_hip.h) followed by
 * the residual add and the next RMSNorm + row quantiser, without the kernel that adds the parts up:
 *   w4a32_matmul_quantized_splitk_parts leaves *parts_out partial products [parts][M][N] in d_scratch (at
 *     least w4a32_splitk_scratch_bytes bytes), each already carrying the row and column factors of the
 *     Linear's output transform; W4A32_ESHAPE when the library does not split this problem;
 *   w4a32_quant_lhs_norm_parts is w4a32_quant_lhs_norm with delta = ((part 0 + part 1) + ...) + bias of
 *     that Linear (d_packed, N_linear = this call's K, K_linear), clamped to the finite f32 range like
 *     every Linear output.
 * Same operators as above (the MLP's down_proj, the decoder layer's residual add and the next layer's
 * input_layer_norm_: modeling_ds_qwen2.hpp:47-54, :175-183); the sum differs from w4a32_matmul_quantized_splitk's
 * in f32 rounding only (the factors are applied before the parts are added instead of after). */
int w4a32_matmul_quantized_splitk_parts(const void* d_ws, const void* d_packed, int M, int K, int N,
                                        void* d_scratch, size_t scratch_bytes, int* parts_out, void* stream);
int w4a32_quant_lhs_norm_parts(const float* d_h, const void* d_parts, int parts, const void* d_packed,
                               int K_linear, const float* d_weight, float eps, float* d_h_out, int M, int K,
                               void* d_ws, void* stream);

/* sin/cos tables [max_pos][head_dim/2]: theta = pos / base^(2d/head_dim).
 * precompute_normal_hf_sin_cos, mllm/Backends/Arm/Kernels/rope.cpp:20-37. */
int w4a32_op_rope_table(float* d_sin, float* d_cos, int max_pos, int head_dim, float base,
                        void* stream);

/* Rotates q [M][n_heads*head_dim] in place, rotates k and copies v [M][n_kv_heads*head_dim] into the
 * caches [n_kv_heads][max_seq][head_dim] at positions pos0 + m. pos0 = *d_pos0 when d_pos0 is not
 * NULL, else the argument. normal_hf_rope (rope.cpp:39-80) + ArmKVCacheOp::forward
 * (mllm/Backends/Arm/Ops/KVCacheOp.cpp:44-72; the reference's head-repeated copies are not stored). */
int w4a32_op_rope_kv(float* d_q, const float* d_k, const float* d_v, const float* d_sin,
                     const float* d_cos, float* d_kcache, float* d_vcache, int M, int n_heads,
                     int n_kv_heads, int head_dim, int max_seq, const int* d_pos0, int pos0,
                     void* stream);

/* im2col of a Conv3D without padding or dilation: d_in [B][C][T][H][W] -> d_out [B*OT*OH*OW][ld_out] with
 * column (c, kt, kh, kw) at c*kt*kh*kw + ..., O* = (size - kernel) / stride + 1; columns from C*kt*kh*kw up
 * to ld_out are written as zeros (pad K to a multiple of 32 and zero-pad the weight rows alike: the
 * convolution is then w4a32_matmul on d_out, as ArmConv3DOp::forward does it,
 * mllm/Backends/Arm/Ops/Conv3DOp.cpp:48-188 with mllm/Backends/Arm/Kernels/conv3d.cpp:15-78). The result
 * rows are [b][ot][oh][ow] x out_channels, i.e. channels-last. */
int w4a32_op_im2col_conv3d(const float* d_in, float* d_out, int B, int C, int T, int H, int W, int kt,
                           int kh, int kw, int st, int sh, int sw, int ld_out, void* stream);

/* Scratch of the decode attention and of argmax: arrival counters + partial results. Must be cleared
 * once with w4a32_op_scratch_init before its first use; the kernels leave it cleared. */
size_t w4a32_op_scratch_bytes(int n_heads);
int w4a32_op_scratch_init(void* d_scratch, int n_heads, void* stream);

/* out[m][h][:] = softmax(q[m][h] . K[0..pos0+m] / sqrt(head_dim)) V, head h reading KV head
 * h / (n_heads / n_kv_heads). head_dim must be 128. With M == 1 and d_scratch given, the keys are split
 * over several wavefronts per head (decode); otherwise one wavefront per (head, query).
 * QWenAttention::forward, modeling_ds_qwen2.hpp:133-151 (matmul, CausalMaskOp.cpp:22-71,
 * SoftmaxOp.cpp:18-50, matmul). */
int w4a32_op_attention(const float* d_q, const float* d_kcache, const float* d_vcache, float* d_out,
                       int M, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                       const int* d_pos0, int pos0, void* d_scratch, void* stream);

/* The same operator for M > 1 rows with scratch lent by the caller: with at least
 * w4a32_op_attention_prefill_scratch_bytes(M, n_heads) bytes at d_part (16-byte aligned; contents need
 * not be kept or cleared) and at most 128 (head, block of 32 queries) pairs, the keys of a query block are
 * dealt to up to 8 workgroups and the last of them to finish combines their results (short prompts, or few
 * rows that continue a long context, would otherwise use a fraction of the CUs; the arrival counters at the
 * head of d_part are cleared by a small launch first); else it runs as w4a32_op_attention does. */
size_t w4a32_op_attention_prefill_scratch_bytes(int M, int n_heads);
int w4a32_op_attention_prefill(const float* d_q, const float* d_kcache, const float* d_vcache,
                               float* d_out, int M, int n_heads, int n_kv_heads, int head_dim,
                               int max_seq, const int* d_pos0, int pos0, void* d_part, size_t part_bytes,
                               void* stream);

/* The same operator for M >= 32 rows at a position the host knows, with both products on the 16-bit matrix
 * pipe at f32 accuracy: every f32 operand is split into three bf16 terms and a product is the six partial
 * products that matter (v_mfma_f32_32x32x16_bf16, f32 accumulation; 2.7 x the rate of the f32 matrix
 * instruction, same exponent range as f32, error below 2^-22 of |x||y| per product). A first launch splits K and V
 * of keys [0, pos0 + M) (V transposed) into d_scratch: at least
 * w4a32_op_attention_prefill_bf16x3_scratch_bytes(pos0 + M, n_kv_heads) bytes, 16-byte aligned, contents need
 * not be kept. Same reference operator as w4a32_op_attention (modeling_ds_qwen2.hpp:133-151). */
size_t w4a32_op_attention_prefill_bf16x3_scratch_bytes(int n_keys, int n_kv_heads);
int w4a32_op_attention_prefill_bf16x3(const float* d_q, const float* d_kcache, const float* d_vcache,
                                      float* d_out, int M, int n_heads, int n_kv_heads, int head_dim,
                                      int max_seq, int pos0, void* d_scratch, size_t scratch_bytes,
                                      void* stream);

/* w4a32_op_rope_kv (position given on the host) followed by w4a32_op_attention_prefill_bf16x3, in two launches
 * instead of three: the launch that splits K and V into bf16 terms also rotates q (in place) and the new rows of
 * k, and appends k and v to the caches. d_q, d_k, d_v are the un-rotated outputs of the q/k/v Linears for rows
 * at positions pos0 .. pos0 + M - 1. Caches, d_q and d_out end up bit-identical to the two operators in
 * sequence. normal_hf_rope (rope.cpp:39-80), ArmKVCacheOp::forward (KVCacheOp.cpp:44-72) and the attention of
 * modeling_ds_qwen2.hpp:133-151. Scratch as for w4a32_op_attention_prefill_bf16x3. */
int w4a32_op_rope_attention_prefill_bf16x3(float* d_q, const float* d_k, const float* d_v, const float* d_sin,
                                           const float* d_cos, float* d_kcache, float* d_vcache, float* d_out,
                                           int M, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                                           int pos0, void* d_scratch, size_t scratch_bytes, void* stream);

/* Decode step (one token at position pos0) with w4a32_op_rope_kv folded into the attention launch:
 * d_q, d_k, d_v are the un-rotated outputs of the q/k/v Linears; the kernel rotates q and k, appends k
 * and v to the caches at pos0 and attends over keys 0..pos0. Same results as the two operators in
 * sequence (d_q itself is left un-rotated). */
int w4a32_op_rope_attention_decode(const float* d_q, const float* d_k, const float* d_v,
                                   const float* d_sin, const float* d_cos, float* d_kcache,
                                   float* d_vcache, float* d_out, int n_heads, int n_kv_heads,
                                   int head_dim, int max_seq, const int* d_pos0, int pos0,
                                   void* d_scratch, void* stream);

/* The same decode step followed by the Linear that reads the attention output (o_proj: K = n_heads *
 * head_dim inputs, N outputs, d_packed from w4a32_quant_pack_rhs), as the decoder's step issues the two:
 * the attention launch leaves its key slices unmerged and the Linear merges them while it loads its input
 * row, so no workgroup of the attention waits for another. d_y [N] receives what
 * w4a32_op_rope_attention_decode followed by w4a32_matmul (M = 1) would, bit for bit; the attention output
 * itself is not materialised. W4A32_ESHAPE when the Linear's shape has no such kernel (K > 3072, or an
 * lm_head-sized N): then call the two operators.
 * Reference: the attention block of modeling_ds_qwen2.hpp:126-153 followed by o_proj (:154). */
int w4a32_op_rope_attention_decode_linear(const float* d_q, const float* d_k, const float* d_v,
                                          const float* d_sin, const float* d_cos, float* d_kcache,
                                          float* d_vcache, const void* d_packed, int N, float* d_y,
                                          int n_heads, int n_kv_heads, int head_dim, int max_seq,
                                          const int* d_pos0, int pos0, void* d_scratch, void* stream);

/* *d_token = index of the first maximum of d_logits[0..n) (AutoLLM.hpp:70-88); when d_pos_to_advance
 * is not NULL, *d_pos_to_advance += 1 afterwards. */
int w4a32_op_argmax(const float* d_logits, int n, void* d_scratch, int64_t* d_token,
                    int* d_pos_to_advance, void* stream);

/* One decode row (M = 1) through 1..4 W4A32 Linears that share it, with the operators around them
 * folded into the same launch:
 *   in front  (d_norm_weight != NULL): row = d_x + d_delta (d_delta may be NULL; the sum is also stored
 *             to d_sum_out when that is not NULL - it must not alias d_x), then RMSNorm with d_norm_weight;
 *   behind    (silu_pair != 0, count == 2, N[0] == N[1]): d_y[0] = silu(linear0) * linear1, d_y[1] unused.
 * The fusions of QWenDecoder::forward / QWenMLP::forward (modeling_ds_qwen2.hpp:47-54,175-183) that cost a
 * launch each when run as separate operators. Returns W4A32_ENOTSUP when the shape does not fit the
 * single-launch kernel (the caller then runs the operators one by one). */
/* Zero-initialise the struct before filling it: fields added at its end (in_parts, out_parts) select other
 * forms of the call when they are not 0. */
typedef struct {
  const float* d_x;
  const float* d_delta;
  float* d_sum_out;
  const float* d_norm_weight;
  float norm_eps;
  int K;
  int count;
  const void* d_packed[4];
  int N[4];
  float* d_y[4];
  int silu_pair;
  int in_parts;   /* 0 or 1: a single row. 2 or 3: the row is given in that many partial rows, K floats apart, which
                     the launch adds up ((r0 + r1) + r2), clamped to the finite f32 range like every Linear
                     output, before it does anything else - at d_delta when
                     d_norm_weight is given (d_delta is then required), else at d_x. Not with silu_pair; for an
                     lm_head-sized Linear (N >= 32768) only as a single Linear with a norm (W4A32_ENOTSUP else). */
  int out_parts;  /* 0 or 1: d_y holds the Linears' outputs. > 1 (count == 1, no norm, no pair, in_parts <= 1;
                     must equal w4a32_decode_kparts(K, N[0])): the Linear's k range is dealt to that many workgroups
                     per tile row and d_y[0] receives [out_parts][N[0]] partial rows whose sum is the output (bias
                     included; the parts themselves are not clamped, a reader that adds them up clamps the sum),
                     for the next w4a32_decode_linear via in_parts. */
} w4a32_decode_linear_args;
int w4a32_decode_linear(const w4a32_decode_linear_args* args, void* stream);

/* Parts into which w4a32_decode_linear would split a [N][K] Linear's k range: 2 for a long K with few output
 * rows (down_proj, K = 8960, N = 1536: its 96 tile rows alone would leave 160 of 256 CUs idle), else 1 (no
 * split). 0 on an invalid shape. No counterpart in the reference, which runs a decode Linear as one task
 * (kai_linear.cpp:366-396). */
int w4a32_decode_kparts(int K, int N);

/* ---- operators of the engine's op-by-op path ------------------------------------------------
 * What the reference's model code dispatches one by one and the decoder runner below fuses away. They exist
 * so that a backend can offer every operator of mllm/Models/ds_qwen2/modeling_ds_qwen2_fa2_fp16.hpp:88-133
 * (activations [B, S, H, D], RoPE layout kBSHD, KV cache layout kBSHD_NO_REPEAT). n % 4 == 0. */

/* out = x / (1 + exp(-x)) (ArmSiLUOp, mllm/Backends/Arm/Ops/SiLUOp.cpp) and out = a * b (ArmMulOp,
 * mllm/Backends/Arm/Ops/ElewiseOps.cpp). SiLU followed by Mul equals w4a32_op_silu_mul bit for bit. */
int w4a32_op_silu(const float* d_x, float* d_out, size_t n, void* stream);
int w4a32_op_mul(const float* d_a, const float* d_b, float* d_out, size_t n, void* stream);

/* y[m][h][:] = RoPE of x[m][h][:] at position pos0 + m, rows [M][n_heads][head_dim] (normal_hf_rope_shd,
 * mllm/Backends/Arm/Kernels/rope.cpp, layout kBSHD); tables as w4a32_op_rope_table builds them, with
 * table_rows rows. d_y may be d_x. */
int w4a32_op_rope(const float* d_x, float* d_y, const float* d_sin, const float* d_cos, int M, int n_heads,
                  int head_dim, int pos0, int table_rows, void* stream);

/* Causal attention with K and V laid out [n_keys][n_kv_heads][head_dim] (the kBSHD_NO_REPEAT cache at batch
 * 1, mllm/Backends/Arm/Ops/KVCacheOp.cpp:74-88): query m at position pos0 + m sees keys 0..pos0 + m.
 * ArmFlashAttn2Op::forward, mllm/Backends/Arm/Ops/FlashAttention2Op.cpp:221-245. head_dim must be 128. */
int w4a32_op_attention_bshd(const float* d_q, const float* d_k, const float* d_v, float* d_out, int M,
                            int n_heads, int n_kv_heads, int head_dim, int n_keys, int pos0, void* stream);

/* C[M][N] = A[M][K] B[N][K]^T, dense f32 (MatMulOp with transpose_b, mllm/Backends/Arm/Ops/MatMulOp.cpp:131-167:
 * how the reference applies lm_head, modeling_ds_qwen2.hpp:209-213). K % 4 == 0. M <= 8 streams B once. */
int w4a32_op_matmul_f32_nt(const float* d_a, const float* d_b, float* d_c, int M, int N, int K, void* stream);

/* Element types of a dense (unquantised) operand. The reference's W4A32 quantizer configuration stores lm_head
 * and the three RMSNorm weights as Fp16 (scripts/QuantCfg/ds_qwen2/1.5B-W4A32-KAI.json:33-45). */
#define W4A32_DENSE_F32 1
#define W4A32_DENSE_F16 2

/* The same product with B [N][K] held as f32 or f16 (b_dtype = W4A32_DENSE_*): an f16 element widens to f32
 * exactly, every product and sum is f32. With K % 8 == 0 and M <= 8, B is streamed once and the f16 and the f32
 * form of the same values give identical bits. K % 4 == 0. */
int w4a32_op_matmul_nt(const float* d_a, const void* d_b, int b_dtype, float* d_c, int M, int N, int K,
                       void* stream);

/* d_out[i] = (float)d_in[i] for n IEEE half values (exact): Fp16 parameters of a model file are widened once at
 * load and the f32 operators run on the result. */
int w4a32_op_f16_to_f32(const void* d_in, float* d_out, size_t n, void* stream);

/* ---- a batch of sequences on a paged cache ------------------------------------------------------
 * Sequences of different lengths share pools of pages: token t of sequence b lies in page
 * d_table[b][t / page] at t % page. A step takes rows of all of them at once: sequence b owns rows
 * d_row_start[b] .. d_row_start[b + 1] (one token, a few drafted ones, a prompt's portion, or none), which
 * stand behind its d_len[b] tokens. Lengths, tables and row starts are device memory: a launch sequence that was
 * captured into a HIP graph serves later steps. Rows behind the last sequence's are left as they are, in every
 * operator (a batch padded to a fixed size).
 *
 * What a device array may say wrongly is kept inside the pools: a page number outside [0, n_pages) stands for a page
 * that is not there (its tokens are not seen and not written; pages that a window has left may be given back so), a
 * negative length is 0 and one past 2^30 is that, tokens behind the table's end are not there (rows that stand behind it see what
 * their windows leave them), and a sequence has at most max_rows rows. Row starts
 * do not decrease; where they do, what the rows get is unspecified.
 *   Sequences may name the same page (a prompt that they share) as long as no call writes it: tokens are appended, and weights
 * added up, only in pages that one sequence names once.
 *
 * The reference has one sequence per model and caches of a fixed length (mllm/Backends/Arm/Ops/KVCacheOp.cpp:44-72). */
#define W4A32_CACHE_F32 1
#define W4A32_CACHE_F16 2
#define W4A32_CACHE_BF16 3
#define W4A32_PAGED_MAX_DIM 256

/* Rows are f32 with any cache, or bf16 with a bf16 cache (`act_bf16`). dim % 8 == 0, dim <= 256; page is a power of two
 * from 16 on; table_ld * page and rows * heads stay below 2^30. Pools and rows on 16 bytes; row strides (ld*, in
 * elements) are multiples of 8 that hold a row. Zero-initialise the structs before filling them. */
typedef struct {
  void *d_k, *d_v;        /* [n_pages][kv_heads][page][dim] of `dtype` */
  float* d_weight;        /* [n_pages][kv_heads][page]: attention weight that each token has received; or NULL */
  const int* d_table;     /* [n_seqs][table_ld] */
  int* d_len;             /* [n_seqs]: tokens a sequence has in the cache, before this step's rows */
  int dtype;              /* W4A32_CACHE_* */
  int n_pages, page, kv_heads, dim, n_seqs, table_ld;
} w4a32_paged_cache;

typedef struct {
  const int* d_row_start;   /* [n_seqs + 1] */
  int rows;                 /* rows the buffers hold: no row number reaches it */
  int max_rows;             /* most rows of one sequence */
  int heads;                /* query heads, a multiple of kv_heads: head h reads kv head h / (heads / kv_heads) */
  int act_bf16;
  const void* d_q;          /* [rows][heads][dim] */
  void* d_out;              /* [rows][heads][dim]: rotated q (append; may be d_q), attention's output (apart from d_q) */
  int ldq, ldo;
} w4a32_paged_rows;

/* q and k of the rows are rotated (dimension i with i + rot_dims / 2, for i < rot_dims / 2; tables
 * [table_rows][rot_dims / 2] as w4a32_op_rope_table builds them), k and v are written behind the sequences' tokens, and
 * the added-up weight of the new tokens is set to 0. d_pos [n_seqs]: the position that a sequence's first row is rotated
 * to (NULL: d_len; they differ once tokens were evicted). d_len stays as it is. rot_dims 0: no rotation (d_sin, d_cos
 * unused). d_q NULL: keys and values alone. Rows at positions outside the tables are left out, as are rows without a slot
 * in a page that is there (their q is rotated all the same). Rotation in f32, one rounding to each stored type.
 * normal_hf_rope (rope.cpp:39-80) and ArmKVCacheOp::forward (KVCacheOp.cpp:44-72) per sequence. */
int w4a32_op_paged_append(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, const void* d_k, int ldk,
                          const void* d_v, int ldv, const int* d_pos, const float* d_sin, const float* d_cos,
                          int rot_dims, int table_rows, void* stream);

/* out = softmax(scale q K^T) V per head over what a row sees: row j of sequence b, which stands at slot s = d_len[b] + j
 * (appended before the call), sees slots t <= s with t > s - window or t < first (window 0: all). A row that sees nothing
 * gets zeros; what is not finite reaches only the rows that see it (a value as in the formula, an infinity of a token with next to no
 * weight too; an infinity in q or in a key may make a row NaN where a score of -infinity would leave the token out). With
 * `accumulate` the weights are added to cache->d_weight: for every cached token the sum over the rows and over the heads of its kv
 * head, in a fixed order (the same call gives the same bits).
 *   Sums, maxima and products are f32 at f32 accuracy for f32 rows (a 16-bit cache's elements are exact operands of the
 * 16-bit matrix instructions, q and the weights enter as two f16 or three bf16 terms); for bf16 rows the weights enter
 * the second product as bf16, as the output is rounded. `scale` is finite. Scores are within f32's range, and so are a row's sums of
 * values, which weigh up to 2^8 each before they are divided: values below 2^100 are safe on any cache.
 *   d_scratch: w4a32_op_paged_attention_scratch_bytes() bytes on 16 bytes, of any contents, for one call at a time (calls that
 * overlap in time, on two streams or in two graphs, need one each). That serves every window; for one window and first, for which
 * less does, ask w4a32_op_paged_attention_window_scratch_bytes(). Both are 0 for a call that w4a32_op_paged_attention refuses (one
 * without a window, the former). With `accumulate` it holds the scores, 4 bytes for each row of a head (rounded up to 16 or
 * 64 of a kv head) and token that the table has room for: a step of more than 1 GiB of them is gone through in passes of 128 rows or
 * more, and with scratch memory for fewer rows at once in more passes (each adds its sums to cache->d_weight).
 * QWenAttention::forward, modeling_ds_qwen2.hpp:133-151, per sequence. */
size_t w4a32_op_paged_attention_scratch_bytes(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows,
                                              int accumulate);
size_t w4a32_op_paged_attention_window_scratch_bytes(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, int window,
                                                     int first, int accumulate);
int w4a32_op_paged_attention(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, float scale, int window,
                             int first, int accumulate, void* d_scratch, size_t scratch_bytes, void* stream);

/* Of every sequence's tokens `budget` stay, per kv head: the first `first` ones, the last `recent` ones and of the others
 * those with the largest added-up weight (of equal ones the earlier; NaN counts as +infinity). Their keys, values and
 * weights go in order to slots 0, 1, .. of the sequence in `to` (same sizes; pages that no table of `cache` names: what is
 * read is not what is written), to->d_len becomes min(length, budget), and d_kept [n_seqs][kv_heads][budget] (int32, or
 * NULL) the slots that stayed, -1 behind them. A sequence within its budget is copied whole. What lies in a page that is
 * not there is lost: as a source it counts with weight 0 and is written as zeros, as a destination it is dropped.
 * first + recent <= budget; both caches have weights. The slots of `to` are the order of the tokens and no longer their
 * positions: give w4a32_op_paged_append d_pos from then on.
 *   d_scratch: w4a32_op_paged_evict_scratch_bytes() bytes on 16 bytes, of any contents, for one call at a time. */
size_t w4a32_op_paged_evict_scratch_bytes(const w4a32_paged_cache* cache, int budget);
int w4a32_op_paged_evict(const w4a32_paged_cache* cache, const w4a32_paged_cache* to, int budget, int first, int recent,
                         int* d_kept, void* d_scratch, size_t scratch_bytes, void* stream);

/* Verification of drafted tokens. Sequence b's rows are its last token and then the tokens drafted behind it (d_tokens
 * [rows]); row r's logits (f32 [rows][ldl]) judge token r + 1. With p = softmax(logits / temperature) and q the draft
 * model's distribution, softmax(d_draft[r] / temperature) (f32 [rows][ldd], a sequence's last row is not read; NULL: the
 * drafted token alone has q = 1), token t is accepted while uniform[r] q(t) < p(t). Behind the last
 * accepted one the next token is drawn: where a token was refused from max(p - q, 0), else from p, as the least index whose
 * running sum exceeds choice[b] times the whole sum. uniform [rows] and choice [n_seqs] are the caller's numbers from
 * [0, 1). temperature 0: a token is accepted where it is the first maximum (which a NaN is not), and the next token is the
 * first maximum, -1 where all are -infinity or NaN (no draft logits or numbers are read; they may be NULL).
 *   d_count[b] = accepted tokens + 1, the rows that stay; d_next[b] = the next token; d_len (may be NULL) += d_count.
 * A sequence without rows gets count 0 and token -1, and a token that has no distribution to come from (no finite
 * logit, a NaN, +infinity) is -1; -infinity is a probability of 0, and a drafted token outside [0, vocab) is refused.
 * Exponentials and sums are held in 64 bits, 1e-11 relative: the choice depends on neither the order of sums nor the sizes of the parts.
 * Per sequence what AutoLLM.hpp:70-88 does for one token, with the test that keeps the target's distribution.
 *   d_scratch: w4a32_op_verify_drafts_scratch_bytes() bytes on 16 bytes, of any contents, for one call at a time. */
typedef struct {
  const float* d_logits;      /* [rows][ldl] */
  const float* d_draft;       /* [rows][ldd], or NULL */
  const int* d_row_start;     /* [n_seqs + 1] */
  const int64_t* d_tokens;    /* [rows] */
  const float *d_uniform, *d_choice;
  int* d_count;               /* [n_seqs] */
  int64_t* d_next;            /* [n_seqs] */
  int* d_len;                 /* [n_seqs], or NULL */
  int rows, max_rows, n_seqs, vocab, ldl, ldd;
  float temperature;
} w4a32_verify_args;
size_t w4a32_op_verify_drafts_scratch_bytes(int rows, int vocab, int n_seqs);
int w4a32_op_verify_drafts(const w4a32_verify_args* args, void* d_scratch, size_t scratch_bytes, void* stream);

/* ---- decoder runner -------------------------------------------------------------------- */

typedef struct {
  int hidden, n_heads, n_kv_heads, head_dim, intermediate, n_layers, vocab;
  int max_seq;           /* KV cache capacity (the reference's max_cache_length) */
  int max_batch_tokens;  /* longest prompt chunk a prefill call may take */
  float rope_theta, rms_eps;
} w4a32_decoder_config;

/* Device pointers; W4 blobs as produced by w4a32_quant_pack_rhs ([N][K] = [out][in]). */
typedef struct {
  const void *q, *k, *v, *o, *gate, *up, *down;
  const float *attn_norm, *ffn_norm;
} w4a32_layer_weights;

/* Zero-initialise the struct before filling it (fields may be added at its end). */
typedef struct {
  const float* embedding;             /* [vocab][hidden] f32 */
  const float* final_norm;            /* [hidden] */
  const void* lm_head;                /* W4 blob [vocab][hidden]; may be NULL when lm_head_dense is given */
  const w4a32_layer_weights* layers;  /* HOST array of n_layers entries */
  /* lm_head as the reference applies it (a dense matmul with transpose_b, modeling_ds_qwen2.hpp:209-213):
   * [vocab][hidden] of lm_head_dense_dtype (W4A32_DENSE_F16 as the reference's quantizer stores it, or
   * W4A32_DENSE_F32). When not NULL it is used instead of lm_head; hidden % 8 == 0. */
  const void* lm_head_dense;
  int lm_head_dense_dtype;
} w4a32_decoder_weights;

/* Bytes of the decoder state (KV caches, activations, tables, counters), 256-byte aligned base. */
size_t w4a32_decoder_state_bytes(const w4a32_decoder_config* cfg);
/* Byte offsets inside the state, for inspection: 0 = position counter (int32), 1 = last logits
 * (f32 [vocab]), 2 = residual stream rows (f32 [max_batch_tokens][hidden]). */
size_t w4a32_decoder_state_offset(const w4a32_decoder_config* cfg, int which);

/* Builds the RoPE tables, clears the counters, position = 0. */
int w4a32_decoder_init(const w4a32_decoder_config* cfg, void* d_state, void* stream);

/* Runs n_tokens prompt tokens at positions pos0.. through the model (QWenForCausalLM::forward,
 * modeling_ds_qwen2.hpp:202-215), leaves the last row's logits in the state, the greedy next token in
 * *d_next_token and the position counter at pos0 + n_tokens. */
int w4a32_decoder_prefill(const w4a32_decoder_config* cfg, const w4a32_decoder_weights* w,
                          void* d_state, const int64_t* d_tokens, int n_tokens, int pos0,
                          int64_t* d_next_token, void* stream);

/* One greedy decode step at the state's current position (AutoLLM generate loop, AutoLLM.hpp:40-66):
 * reads *d_token_in, writes *d_token_out (may be the same address), advances the position. The launch
 * sequence does not depend on the position: capture it once, replay it per token. The caller keeps
 * the position below max_seq: the step itself cannot refuse (the position is device memory, and a replayed
 * graph never returns to the host). A step issued at position >= max_seq stays inside the cache - the
 * attention treats the position as max_seq - 1 and overwrites the last row - but its token is meaningless
 * and the counter keeps advancing; w4a32_decoder_prefill, whose pos0 is a host argument, returns W4A32_ESHAPE
 * when pos0 + n_tokens exceeds max_seq. */
int w4a32_decoder_step(const w4a32_decoder_config* cfg, const w4a32_decoder_weights* w, void* d_state,
                       const int64_t* d_token_in, int64_t* d_token_out, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* W4A32_DECODER_H */
