/*
 * trinix_b200 — C ABI of the sm_100a (B200) backend for Trinix's layer hot path: the forward of
 * the norms, int8 ops, RoPE, GLUs and attention, and the backward of the norms, GLUs and RoPE.
 *
 * Every entry point is `extern "C"`, takes plain device pointers, sizes and
 * strides (in ELEMENTS unless a name ends in `_bytes`), enqueues work on the
 * given CUDA stream and returns a status code (0 = ok, < 0 = error). Nothing
 * here allocates device memory, synchronises the stream or throws. Arguments
 * are validated before any launch; an error code means nothing was launched.
 * The caller owns every buffer and selects the device (cudaSetDevice) first.
 *
 * Each declaration names the interface of the reference (Trinix 0.1.4, paths
 * relative to its repository root) whose device work it replaces.
 */
#ifndef TRINIX_B200_H_
#define TRINIX_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TRX_ABI_VERSION 1

typedef enum trx_status {
  TRX_OK = 0,
  TRX_ERR_NULL_POINTER = -1,  /* a required pointer is NULL */
  TRX_ERR_DTYPE = -2,         /* dtype code not supported by this entry point */
  TRX_ERR_SHAPE = -3,         /* negative / zero / inconsistent sizes */
  TRX_ERR_ALIGNMENT = -4,     /* pointer or stride not aligned as required */
  TRX_ERR_STRIDE = -5,        /* stride smaller than the extent it spans */
  TRX_ERR_UNSUPPORTED = -6,   /* legal request this build cannot serve (e.g. head_dim) */
  TRX_ERR_CUDA = -7,          /* the CUDA runtime/driver reported an error at launch */
  TRX_ERR_DEVICE_STATUS = -8, /* a kernel recorded a bounded-wait timeout in its status word */
  TRX_ERR_WORKSPACE = -9      /* workspace missing or too small */
} trx_status;

typedef enum trx_dtype { TRX_F32 = 0, TRX_F16 = 1, TRX_BF16 = 2 } trx_dtype;

typedef enum trx_glu_act {
  TRX_GLU_SWIGLU = 0,     /* up * silu(gate) */
  TRX_GLU_GEGLU_TANH = 1, /* up * gelu_tanh(gate) */
  TRX_GLU_REGLU = 2       /* up * max(gate, 0) */
} trx_glu_act;

/* Activation fused behind RMSNorm (trx_rmsnorm_act_fwd). */
typedef enum trx_row_act {
  TRX_ACT_MISH = 0,         /* n * tanh(softplus(n)) */
  TRX_ACT_QUICKGELU = 1,    /* n * sigmoid(1.702 n) */
  TRX_ACT_SQUARED_RELU = 2  /* max(n, 0)^2 */
} trx_row_act;

/* Norm of a query's or key's row (trx_qk_norm_rope_fwd). */
typedef enum trx_norm {
  TRX_NORM_RMS = 0,  /* x rsqrt(mean x^2 + eps) */
  TRX_NORM_LAYER = 1 /* (x - mean) rsqrt(mean (x - mean)^2 + eps) */
} trx_norm;

/* ABI version of the loaded library (TRX_ABI_VERSION at build time). */
int trx_version(void);

/* Static, human-readable text for a status code. */
const char* trx_status_string(int code);

/*
 * RMSNorm forward over R rows of C columns:
 *   rstd = 1/sqrt(mean(x^2) + eps);  y = round_x(w * round_x(x * rstd))
 * (the two roundings to the activation dtype follow the reference's PyTorch
 * backend, trinix/layers/norm/rmsnorm.py:70-75). `rstd_or_null` receives the
 * fp32 per-row rstd when non-NULL.
 * Replaces the launch made by TritonRMSNormFunction.forward,
 * trinix/kernels/rmsnorm_kernel.py:238-269 (kernel :9-61), reached through
 * TritonRMSNormKernel.apply, trinix/kernels/rmsnorm_kernel.py:387-389.
 */
int trx_rmsnorm_fwd(const void* x, const void* w, void* y, float* rstd_or_null, int64_t R,
                    int64_t C, int64_t x_row_stride, int64_t y_row_stride, float eps, int x_dtype,
                    int w_dtype, void* stream);

/*
 * LayerNorm forward: y = (x - mean) * rstd * w + b with biased variance.
 * `w_or_null` / `b_or_null` may be NULL (elementwise_affine=False,
 * trinix/layers/norm/layernorm.py:54-55); both share `wb_dtype`.
 * Replaces TritonLayerNormFunction.forward, trinix/kernels/layernorm_kernel.py:224-353
 * (kernel :11-67), reached through TritonLayerNormKernel.apply, :418-422.
 */
int trx_layernorm_fwd(const void* x, const void* w_or_null, const void* b_or_null, void* y,
                      float* mean_or_null, float* rstd_or_null, int64_t R, int64_t C,
                      int64_t x_row_stride, int64_t y_row_stride, float eps, int x_dtype,
                      int wb_dtype, void* stream);

/*
 * Per-row symmetric int8 quantisation:
 *   scale[r] = max|x[r,:]| / 127 (fp32, IEEE division)
 *   code     = clamp(round_half_even(x / scale), -127, 127); zero rows -> scale 0, codes 0.
 * No counterpart in the reference (it has no int8 code); the contract is the
 * "per-row symmetric int8 quantize/dequantize" configuration of this project's baseline.
 */
int trx_quant_rowwise_i8(const void* x, int8_t* codes, float* scales, int64_t R, int64_t C,
                         int64_t x_row_stride, int64_t codes_row_stride, int x_dtype,
                         void* stream);

/*
 * Inverse of trx_quant_rowwise_i8: y = round_y(float(code) * scale[r]).
 * No counterpart in the reference.
 */
int trx_dequant_rowwise_i8(const int8_t* codes, const float* scales, void* y, int64_t R, int64_t C,
                           int64_t codes_row_stride, int64_t y_row_stride, int y_dtype,
                           void* stream);

/*
 * Fused RMSNorm -> int8: quantises exactly the rows trx_rmsnorm_fwd would
 * write (after rounding to the activation dtype) without writing them.
 * No counterpart in the reference; its structure (norm, then an epilogue on
 * the row held on chip) is that of fused_rmsnorm_activation_forward_kernel,
 * trinix/kernels/fused/rmsnorm_activation_kernel.py:9-77.
 */
int trx_rmsnorm_quant_i8(const void* x, const void* w, int8_t* codes, float* scales, int64_t R,
                         int64_t C, int64_t x_row_stride, int64_t codes_row_stride, float eps,
                         int x_dtype, int w_dtype, void* stream);

/*
 * act(RMSNorm(x)): n = round(w * round(x * rstd)) as trx_rmsnorm_fwd computes it (the product is
 * rounded to the activation dtype only when w has that dtype; any other w dtype leaves it in
 * fp32, PyTorch's promotion), then y = round(act(n)), act one of TRX_ACT_*. One pass over HBM
 * instead of two.
 * Follows FastFusedRMSNormActivation._pytorch_forward,
 * trinix/layers/fused/rmsnorm_activation.py:72-86; replaces
 * TritonFusedRMSNormActivationKernel.apply, trinix/kernels/fused/rmsnorm_activation_kernel.py
 * (kernel :9-77).
 */
int trx_rmsnorm_act_fwd(const void* x, const void* w, void* y, int64_t R, int64_t C,
                        int64_t x_row_stride, int64_t y_row_stride, float eps, int act,
                        int x_dtype, int w_dtype, void* stream);

/*
 * Fused residual add + RMSNorm: s = float(x) + float(residual) (kept in fp32 on chip),
 *   y = round_x(w * round_x(s * rstd(s))); `sum_out_or_null` receives round_x(s), the new
 *   residual stream, when non-NULL.
 * Follows FastFusedResidualRMSNorm._pytorch_forward, trinix/layers/fused/residual_rmsnorm.py:66-73.
 * Replaces TritonFusedResidualRMSNormFunction.forward,
 * trinix/kernels/fused/residual_rmsnorm_kernel.py:212-248 (kernel :9-73), reached through
 * TritonFusedResidualRMSNormKernel.apply(X, Residual, W, eps).
 */
int trx_residual_rmsnorm_fwd(const void* x, const void* residual, const void* w, void* y,
                             void* sum_out_or_null, float* rstd_or_null, int64_t R, int64_t C,
                             int64_t x_row_stride, int64_t res_row_stride, int64_t y_row_stride,
                             int64_t sum_row_stride, float eps, int x_dtype, int w_dtype,
                             void* stream);

/*
 * Fused residual add + LayerNorm: s = float(x) + float(residual) (fp32, on chip),
 *   y = round(round(w * round((s - mean(s)) * rstd)) + b)  — the normalised value is cast to the
 *   activation dtype before the affine part, which runs in the parameters' dtype (a parameter
 *   dtype other than the activation's promotes to fp32 and rounds once at the end);
 *   sum_out_or_null receives round(s). w and b may be NULL.
 * Follows FastFusedResidualLayerNorm._pytorch_forward,
 * trinix/layers/fused/residual_layernorm.py:66-73; replaces
 * TritonFusedResidualLayerNormKernel.apply, trinix/kernels/fused/residual_layernorm_kernel.py
 * (kernel :9-79).
 */
int trx_residual_layernorm_fwd(const void* x, const void* residual, const void* w_or_null,
                               const void* b_or_null, void* y, void* sum_out_or_null,
                               float* mean_or_null, float* rstd_or_null, int64_t R, int64_t C,
                               int64_t x_row_stride, int64_t res_row_stride, int64_t y_row_stride,
                               int64_t sum_row_stride, float eps, int x_dtype, int w_dtype,
                               void* stream);

/*
 * Fused residual add + RMSNorm -> int8: quantises exactly the rows trx_residual_rmsnorm_fwd
 * would write, without writing them; optionally writes the summed residual stream.
 * No counterpart in the reference (it has no int8 code).
 */
int trx_residual_rmsnorm_quant_i8(const void* x, const void* residual, const void* w, int8_t* codes,
                                  float* scales, void* sum_out_or_null, int64_t R, int64_t C,
                                  int64_t x_row_stride, int64_t res_row_stride,
                                  int64_t codes_row_stride, int64_t sum_row_stride, float eps,
                                  int x_dtype, int w_dtype, void* stream);

/*
 * Rotary position embedding, half-split ("rotate_half") form, q and k in one launch:
 *   o[..., :D/2] = x1*cos - x2*sin ;  o[..., D/2:] = x2*cos + x1*sin
 * with cos/sin rows indexed by the sequence position (tables are (S, >= D/2),
 * only the first D/2 columns are read). Tensors are (B, S, H, D) with D
 * contiguous; q and k may have different head counts and arbitrary b/s/h strides.
 * `table_dtype` is TRX_F32 or equal to `x_dtype`; in the latter case every
 * intermediate product is rounded to `x_dtype` like the reference's PyTorch path
 * (trinix/layers/embeddings/rope.py:111-118). `inverse != 0` negates sin.
 * Replaces TritonRoPEFunction.forward, trinix/kernels/rope_kernel.py:165-170
 * (two launches of _rope_rotation_kernel, :11-88), reached through
 * TritonRoPEKernel.apply, :209-213.
 */
int trx_rope_fwd(const void* q, const void* k, const void* cos_table, const void* sin_table,
                 void* q_out, void* k_out, int64_t B, int64_t S, int64_t Hq, int64_t Hk, int64_t D,
                 const int64_t q_strides[3], const int64_t k_strides[3],
                 const int64_t qo_strides[3], const int64_t ko_strides[3],
                 int64_t table_row_stride, int table_dtype, int x_dtype, int inverse,
                 void* stream);

/*
 * Norm of every query's and key's row of D values, with weight w and (TRX_NORM_LAYER only, NULL: none) bias b,
 * and the rotation of trx_rope_fwd, q and k in one launch: y = rotate(norm(x) w + b) with norm_first != 0,
 * else y = norm(rotate(x)) w + b. All arithmetic is fp32, rounded once. D is even and at most 512, tensors are
 * (B, S, H, D) with D contiguous. Row r of the tables (table_rows, >= D/2) has the angles of position r;
 * a token's position is positions[b, s] (int32, or int64 with positions_64 != 0), without positions its index
 * s. A position outside the tables makes its rows NaN. `table_dtype` is TRX_F32 or `x_dtype`; `w_dtype`, of
 * weights and biases, is any. `strides`: (batch, seq, head) of q, k, q_out, k_out, (batch, seq) of positions.
 * Replaces the sequence of trinix/layers/embeddings/rope.py:83-134 and the q / k norm modules in
 * trinix/layers/attention/grouped_query_attention.py:167-178.
 */
int trx_qk_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                         const void* q_bias_or_null, const void* k_bias_or_null, const void* cos_table,
                         const void* sin_table, const void* positions_or_null, void* q_out, void* k_out,
                         int64_t B, int64_t S, int64_t Hq, int64_t Hk, int64_t D, const int64_t strides[14],
                         int64_t table_rows, int64_t table_row_stride, float eps, int norm, int norm_first,
                         int positions_64, int table_dtype, int w_dtype, int x_dtype, void* stream);

/*
 * Gradients of trx_qk_norm_rope_fwd: dq_out / dk_out are those of its outputs, dq / dk (contiguous in D) the
 * inputs'. Those of the weights and biases, in `w_dtype`, are summed in fp32 in an order fixed by the sizes and
 * the device; NULL: not asked for. `strides`: (batch, seq, head) of dq_out, dk_out, q, k, dq, dk,
 * (batch, seq) of positions. The workspace is 16-byte aligned and holds nothing between calls.
 */
int trx_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k,
                         const void* q_weight, const void* k_weight, const void* cos_table,
                         const void* sin_table, const void* positions_or_null, void* dq, void* dk,
                         void* dq_weight_or_null, void* dk_weight_or_null, void* dq_bias_or_null,
                         void* dk_bias_or_null, int64_t B, int64_t S, int64_t Hq, int64_t Hk, int64_t D,
                         const int64_t strides[20], int64_t table_rows, int64_t table_row_stride, float eps,
                         int norm, int norm_first, int positions_64, int table_dtype, int w_dtype,
                         int x_dtype, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of that workspace on the current device; 0 for a head_dim that is refused. */
size_t trx_qk_norm_rope_bwd_workspace_bytes(int64_t D);

/*
 * Gated linear unit forward: y[r, c] = up[r, c] * act(gate[r, c]) for R rows of H columns.
 * `up` and `gate` are separate pointers with their own row strides so that both the
 * reference's concatenated layout (x[..., :H] = up, x[..., H:] = gate) and
 * separate tensors work.
 * Replaces TritonSwiGLUFunction.forward (trinix/kernels/swigelu_kernel.py:121-152),
 * the GeGLU forward (trinix/kernels/geglu_kernel.py:9-49) and the ReGLU forward
 * (trinix/kernels/reglu_kernel.py:9-41), reached through Triton{SwiGLU,GeGLU,ReGLU}Kernel.apply.
 */
int trx_glu_fwd(const void* up, const void* gate, void* y, int64_t R, int64_t H,
                int64_t up_row_stride, int64_t gate_row_stride, int64_t y_row_stride, int act,
                int dtype, void* stream);

/*
 * Backward of the GLUs: dup = dy * act(gate), dgate = dy * up * act'(gate), fp32 math, one
 * rounding per output. Every tensor has its own row stride, so dup / dgate may be the two halves
 * of a concatenated (R, 2H) gradient.
 * Replaces TritonSwiGLUFunction.backward (trinix/kernels/swigelu_kernel.py:154-180, kernel
 * :47-91) and the GeGLU / ReGLU backward kernels (trinix/kernels/geglu_kernel.py:53-108,
 * trinix/kernels/reglu_kernel.py:45-87).
 */
int trx_glu_bwd(const void* dy, const void* up, const void* gate, void* dup, void* dgate,
                int64_t R, int64_t H, int64_t dy_row_stride, int64_t up_row_stride,
                int64_t gate_row_stride, int64_t dup_row_stride, int64_t dgate_row_stride, int act,
                int dtype, void* stream);

/*
 * Bytes of device workspace the norm backward entry points need for R rows of C columns: two
 * (P, C) fp32 blocks of per-CTA column sums (P <= 1024, bounded so a block stays <= 16 MiB) plus
 * (R, 2) fp32 row statistics. Contents on entry are irrelevant; nothing is kept between calls.
 */
size_t trx_norm_bwd_workspace_bytes(int64_t R, int64_t C);

/*
 * RMSNorm backward. With n = x * rsqrt(mean(x^2) + eps) (recomputed from x, nothing saved by the
 * forward is needed) and g = dy * w:  dx = rstd * (g - n * mean(g * n)),  dw = sum_rows dy * n
 * (fp32 sums in a fixed order: deterministic for a given shape and device; stored in w_dtype).
 * dw_or_null == NULL skips the weight gradient.
 * Replaces TritonRMSNormFunction.backward (trinix/kernels/rmsnorm_kernel.py:270-321; kernels
 * rmsnorm_backward_dx_fused :65-147 with its lock-guarded accumulation, rmsnorm_backward_dw
 * :151-194).
 */
int trx_rmsnorm_bwd(const void* dy, const void* x, const void* w, void* dx, void* dw_or_null,
                    int64_t R, int64_t C, int64_t dy_row_stride, int64_t x_row_stride,
                    int64_t dx_row_stride, float eps, int x_dtype, int w_dtype, void* workspace,
                    size_t workspace_bytes, void* stream);

/*
 * LayerNorm backward. n = (x - mean) * rstd, g = dy * w (w == NULL: g = dy):
 *   dx = rstd * (g - mean(g) - n * mean(g * n)),  dw = sum_rows dy * n,  db = sum_rows dy.
 * dw_or_null / db_or_null == NULL skip that gradient.
 * Replaces TritonLayerNormFunction.backward (trinix/kernels/layernorm_kernel.py:298-353; kernels
 * layernorm_backward_dx_fused :71-164, layernorm_backward_dwdb :168-221).
 */
int trx_layernorm_bwd(const void* dy, const void* x, const void* w_or_null, void* dx,
                      void* dw_or_null, void* db_or_null, int64_t R, int64_t C,
                      int64_t dy_row_stride, int64_t x_row_stride, int64_t dx_row_stride, float eps,
                      int x_dtype, int wb_dtype, void* workspace, size_t workspace_bytes,
                      void* stream);

/*
 * Backward of the residual forms: the normalised row is the fp32 sum x + residual, exactly as in
 * trx_residual_rmsnorm_fwd / trx_residual_layernorm_fwd; d/dx and d/dresidual are the same tensor,
 * written once to dx. Otherwise as trx_rmsnorm_bwd / trx_layernorm_bwd (same workspace).
 * Replace TritonFusedResidualRMSNormFunction.backward
 * (trinix/kernels/fused/residual_rmsnorm_kernel.py:251-303; kernels :77-205) and
 * TritonFusedResidualLayerNormFunction.backward
 * (trinix/kernels/fused/residual_layernorm_kernel.py:278-335; kernels :83-225).
 */
int trx_residual_rmsnorm_bwd(const void* dy, const void* x, const void* residual, const void* w,
                             void* dx, void* dw_or_null, int64_t R, int64_t C,
                             int64_t dy_row_stride, int64_t x_row_stride, int64_t res_row_stride,
                             int64_t dx_row_stride, float eps, int x_dtype, int w_dtype,
                             void* workspace, size_t workspace_bytes, void* stream);
int trx_residual_layernorm_bwd(const void* dy, const void* x, const void* residual,
                               const void* w_or_null, void* dx, void* dw_or_null, void* db_or_null,
                               int64_t R, int64_t C, int64_t dy_row_stride, int64_t x_row_stride,
                               int64_t res_row_stride, int64_t dx_row_stride, float eps,
                               int x_dtype, int wb_dtype, void* workspace, size_t workspace_bytes,
                               void* stream);

/*
 * Backward of (residual) RMSNorm / LayerNorm with the forward's row statistics instead of
 * recomputed ones: rstd (and mean) are the fp32 [R] outputs of trx_rmsnorm_fwd,
 * trx_residual_rmsnorm_fwd, trx_layernorm_fwd or trx_residual_layernorm_fwd on the same rows.
 * res_or_null is the residual of the residual forms. Otherwise as trx_rmsnorm_bwd /
 * trx_layernorm_bwd (same workspace, same results up to the statistics' last bits). Replaces nothing
 * beyond what those two replace.
 */
int trx_rmsnorm_bwd_saved(const void* dy, const void* x, const void* res_or_null, const void* w,
                          const float* rstd, void* dx, void* dw_or_null, int64_t R, int64_t C,
                          int64_t dy_row_stride, int64_t x_row_stride, int64_t res_row_stride,
                          int64_t dx_row_stride, int x_dtype, int w_dtype, void* workspace,
                          size_t workspace_bytes, void* stream);
int trx_layernorm_bwd_saved(const void* dy, const void* x, const void* res_or_null,
                            const void* w_or_null, const float* mean, const float* rstd, void* dx,
                            void* dw_or_null, void* db_or_null, int64_t R, int64_t C,
                            int64_t dy_row_stride, int64_t x_row_stride, int64_t res_row_stride,
                            int64_t dx_row_stride, int x_dtype, int wb_dtype, void* workspace,
                            size_t workspace_bytes, void* stream);

/*
 * Backward of act(RMSNorm(x)) (trx_rmsnorm_act_fwd): with z = w * n the upstream gradient becomes
 * dy * act'(z), then as trx_rmsnorm_bwd (same workspace). act is one of TRX_ACT_*.
 * Replaces TritonFusedRMSNormActivationFunction.backward
 * (trinix/kernels/fused/rmsnorm_activation_kernel.py:280-330; kernels :81-233).
 */
int trx_rmsnorm_act_bwd(const void* dy, const void* x, const void* w, void* dx, void* dw_or_null,
                        int64_t R, int64_t C, int64_t dy_row_stride, int64_t x_row_stride,
                        int64_t dx_row_stride, float eps, int act, int x_dtype, int w_dtype,
                        void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of zero-initialised device workspace trx_attn_fwd needs (status word + scheduler state). */
size_t trx_attn_workspace_bytes(void);

/*
 * Attention forward, softmax(scale * Q K^T + bias) V with online softmax:
 *   q (B, Sq, Hq, D), k/v (B, Sk, Hk, D), out (B, Sq, Hq, D); D contiguous, D in {64, 128};
 *   Hq % Hk == 0, query head h reads kv head h / (Hq / Hk)  (GQA / MQA natively; a kv head
 *   stride of 0 — an expanded single head — is accepted);
 *   causal: key j visible to query i iff j <= i;
 *   window_left/right >= 0: visible iff -left <= j - i <= right (pass -1/-1 for no window);
 *   slopes_or_null: fp32 [Hq], adds -slope[h] * |i - j| after scaling (ALiBi);
 *   lse_or_null: fp32 (B, Hq, Sq) natural-log sum-exp per row, optional.
 * `workspace` points at trx_attn_workspace_bytes() bytes that were zero when first used;
 * word 0 accumulates a non-zero code if a bounded on-chip wait ever gave up.
 * strides are (batch, seq, head) in elements. dtype: TRX_BF16 or TRX_F16.
 * Replaces TritonAttentionKernel.apply, trinix/kernels/attention_kernel.py:498-664
 * (kernel _fwd_kernel, :235-434), reached through triton_attn_func,
 * trinix/layers/attention/functional.py:8-140, and the flash_attn_func call at
 * trinix/layers/attention/base.py:338-344.
 */
int trx_attn_fwd(const void* q, const void* k, const void* v, void* out, float* lse_or_null,
                 const float* slopes_or_null, int64_t B, int64_t Sq, int64_t Sk, int64_t Hq,
                 int64_t Hk, int64_t D, const int64_t q_strides[3], const int64_t k_strides[3],
                 const int64_t v_strides[3], const int64_t o_strides[3], float scale, int causal,
                 int64_t window_left, int64_t window_right, int dtype, void* workspace,
                 size_t workspace_bytes, void* stream);

/*
 * trx_attn_fwd with a dense additive mask: softmax(scale * Q K^T + mask [+ ALiBi]) V.
 *   mask: (B, Hq, Sq, Sk) values added to the scaled scores (0 keeps, -inf hides); fp32 or the
 *   activation dtype (mask_dtype); mask_strides = (batch, head, query) in elements, the key
 *   stride is 1; a batch or head stride of 0 broadcasts, which is how the reference's 2-D
 *   (Sq, Sk), 3-D (B, Sq, Sk) and 4-D (B, 1, Sq, Sk) masks are passed without expanding them.
 *   causal / window / ALiBi combine with it; a row whose keys are all hidden returns 0.
 * Every KV tile a query tile can see is visited (a dense mask gives no tile to skip), and the
 * mask is read once per score: 4 bytes per score for fp32, so the call is bound by the mask's
 * HBM traffic unless the mask is broadcast over batch and heads.
 * Replaces the attn_mask path of TritonAttentionKernel.apply,
 * trinix/kernels/attention_kernel.py:479-495 (_prepare_mask) and :9-231 (_fwd_kernel_with_mask);
 * mask semantics of FastBaseAttention._apply_pytorch_attention,
 * trinix/layers/attention/base.py:381-392.
 */
int trx_attn_fwd_mask(const void* q, const void* k, const void* v, void* out, float* lse_or_null,
                      const float* slopes_or_null, const void* mask, int mask_dtype,
                      const int64_t mask_strides[3], int64_t B, int64_t Sq, int64_t Sk, int64_t Hq,
                      int64_t Hk, int64_t D, const int64_t q_strides[3],
                      const int64_t k_strides[3], const int64_t v_strides[3],
                      const int64_t o_strides[3], float scale, int causal, int64_t window_left,
                      int64_t window_right, int dtype, void* workspace, size_t workspace_bytes,
                      void* stream);

/*
 * trx_attn_fwd_mask with dropout on the attention probabilities (mask_or_null may be NULL):
 *   out = sum_j keep_ij * P_ij / (1 - p_eff) * V_j,   P = softmax(scale * Q K^T + bias)
 * i.e. the probabilities are normalised first and dropped afterwards, the order of the reference's
 * PyTorch backend (F.dropout on the softmax output, trinix/layers/attention/base.py:394-397); the
 * LSE output is that of the undropped scores. The keep decision of element (b, h, i, j) is a pure
 * function of (seed, offset, b, h, i, j): byte (j mod 16) of Philox4x32-10 with key
 * (seed & 0xffffffff, seed >> 32) and counter (j / 16, i, b * Hq + h, offset), little-endian over
 * the four result words; the element is dropped when that byte is below
 * t = clamp(round(256 * dropout_p), 1, 255), so the realised probability is p_eff = t / 256 and
 * kept elements are scaled by 256 / (256 - t). The stream can therefore be rebuilt on the host,
 * which is how the tests check it element for element. 0 <= dropout_p < 1; 0 means no dropout.
 * Replaces the dropout branch of the reference's kernel, trinix/kernels/attention_kernel.py:395-405
 * (seed drawn at :526-532), whose own random stream (Triton's tl.rand) cannot be reproduced and
 * whose normaliser, unlike its PyTorch backend's, includes the dropped probabilities.
 */
int trx_attn_fwd_dropout(const void* q, const void* k, const void* v, void* out,
                         float* lse_or_null, const float* slopes_or_null, const void* mask_or_null,
                         int mask_dtype, const int64_t mask_strides[3], int64_t B, int64_t Sq,
                         int64_t Sk, int64_t Hq, int64_t Hk, int64_t D, const int64_t q_strides[3],
                         const int64_t k_strides[3], const int64_t v_strides[3],
                         const int64_t o_strides[3], float scale, int causal, int64_t window_left,
                         int64_t window_right, int dtype, float dropout_p, uint64_t seed,
                         uint32_t offset, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Attention over packed sequences: q (Tq, Hq, D), k / v (Tk, Hk, D), out (Tq, Hq, D), D contiguous, D in
 * {64, 128}, strides (row, head) in elements. Sequence s of n_seq has the rows cu_q[s] .. cu_q[s + 1] - 1
 * and the keys cu_k[s] .. cu_k[s + 1] - 1 (device memory, n_seq + 1 ascending values each, the first 0;
 * a value out of range or out of order is cut to what the tensors hold: such a call's results are
 * undefined, its accesses are not). With Sq rows and Sk keys, query i stands at key position
 * i + Sk - Sq: causal, window and ALiBi of trx_attn_fwd are relative to that, so a whole prompt
 * (Sq == Sk), a piece of one behind cached keys and a single token (Sq == 1) need nothing else. A row
 * without a visible key returns 0 (LSE -inf).
 *   lse_or_null: fp32 (Hq, Tq);
 *   max_sq: no sequence has more rows (0: unknown). Up to 16 selects the kernel for few rows, which does the
 *     first max_sq rows of a longer sequence, as rows of the whole of it, and leaves the others unwritten;
 *   zero_rest: rows behind cu_q[n_seq] are written as rows without a visible key; otherwise not touched.
 * Keys outside a sequence are never used, whatever their values (NaN among them).
 * `workspace` as for trx_attn_fwd. No counterpart in the reference, whose attention takes one batch of
 * equal lengths (trinix/kernels/attention_kernel.py:498-664) and has prompts of different lengths padded.
 */
int trx_attn_fwd_packed(const void* q, const void* k, const void* v, void* out, float* lse_or_null,
                        const float* slopes_or_null, const int32_t* cu_q, const int32_t* cu_k,
                        int64_t n_seq, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                        const int64_t q_strides[2], const int64_t k_strides[2],
                        const int64_t v_strides[2], const int64_t o_strides[2], float scale, int causal,
                        int64_t window_left, int64_t window_right, int64_t max_sq, int zero_rest,
                        int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Attention for a batch that shares a prefix: the prefix's keys and values (P, Hk, D), strides (row, head),
 * are those of every sequence, in front of its own (B, S, Hk, D), strides (batch, row, head), of which
 * lengths[b] (device memory, cut to 0 .. S; NULL: S) are in use; the others are never used, whatever their
 * values (NaN among them). q, out (B, Sq, Hq, D): the last Sq tokens of each sequence. Over the P + lengths[b]
 * keys of the concatenation this is causal attention of trx_attn_fwd_packed: query i stands at
 * P + lengths[b] - Sq + i and sees the keys up to there; slopes_or_null (ALiBi) counts from there.
 * scale >= 1e-30. lse_or_null: fp32 (B, Hq, Sq). TRX_ERR_SHAPE beyond B, Hq = 65535, B * Sq = 2^30,
 * P, S = 2^29, Sq = 65535 * 256.
 * With few rows to a sequence, or a long prefix, the prefix is read and computed once for all sequences, its
 * keys split over the GPU (a choice by sizes alone); the splits' results need `parts`:
 * trx_attn_shared_bytes(...) bytes of device memory, asked for with the call's device current, 16-byte
 * aligned (0: none, parts may be NULL), contents on entry irrelevant, nothing kept between calls. It wants
 * the batch's rows evenly spaced (q_strides[0] == Sq * q_strides[1]); others take one pass, whatever it costs.
 * `workspace` as for trx_attn_fwd. No counterpart in the reference, whose attention takes one batch
 * (trinix/kernels/attention_kernel.py:498-664) and has the prefix repeated for every sequence.
 */
size_t trx_attn_shared_bytes(int64_t B, int64_t Sq, int64_t P, int64_t S, int64_t Hq, int64_t Hk,
                             int64_t D);
int trx_attn_fwd_shared(const void* q, const void* prefix_k, const void* prefix_v, const void* k,
                        const void* v, void* out, float* lse_or_null, const float* slopes_or_null,
                        const int32_t* lengths_or_null, int64_t B, int64_t Sq, int64_t P, int64_t S,
                        int64_t Hq, int64_t Hk, int64_t D, const int64_t q_strides[3],
                        const int64_t pk_strides[2], const int64_t pv_strides[2],
                        const int64_t k_strides[3], const int64_t v_strides[3],
                        const int64_t o_strides[3], float scale, int dtype, void* parts,
                        size_t parts_bytes, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Status word of an attention workspace, read without synchronising. `host_word` is host
 * memory the caller keeps alive across calls (pinned memory keeps the copy asynchronous),
 * zero before the first call. If *host_word — as copied there by an earlier call — is already
 * non-zero, a kernel gave up on a bounded wait and every later launch on that workspace has
 * skipped its work: the call returns TRX_ERR_DEVICE_STATUS and enqueues nothing; the caller
 * zeroes the device word and *host_word before using the workspace again. Otherwise a 4-byte
 * copy of the device word into *host_word is enqueued on `stream`, behind the launches already
 * there. Call it after each trx_attn_fwd / trx_attn_fwd_mask (or every few).
 * Replaces nothing in the reference: there the failure path is the silent PyTorch fallback of
 * trinix/layers/attention/base.py:435-439.
 */
int trx_attn_status(const void* workspace, unsigned int* host_word, void* stream);

/*
 * A cache of keys and values in pages, and a batch's place in it. `k_pages` / `v_pages` are (pages, Hk,
 * page_size, D) of the activation type, or, with scales, (pages, Hk, page_size, D / 2) bytes of two 4-bit codes
 * each (column 2 j of a row low, 2 j + 1 high) with scales (pages, Hk, page_size, 2) of fp32 (step, lowest):
 * a value is lowest + code * step; a row's lowest value has code 0, its highest 15, the others the nearest
 * (halfway: the even one), step is (highest - lowest) * fp32(1/15). A row whose values are within 2^-76 of each
 * other has step 0 and codes 0; one with a value that is not finite, or that spans more than 2^120, has both
 * numbers NaN. D is 64 or 128, page_size a multiple of 16 up to 4096. Position p of sequence b is row
 * p % page_size of page block_table[b][p / page_size] of (n_seq, width); numbers outside [0, pages) name no page:
 * nothing is written there and rows of zeros are read. Strides: (page, head, row) of k_pages, v_pages in elements
 * (codes: bytes, rows contiguous), (page, head) of k_scales, v_scales, the row of block_table: 11 in this order,
 * the last in each entry's `strides`. Bases are 16-byte aligned and strides multiples of 16 bytes.
 * No counterparts in the reference, whose cache is a concatenation for each step
 * (trinix/layers/attention/grouped_query_attention.py:178-184).
 */

/*
 * Append: n_seq sequences of S new tokens each (k, v (n_seq, S, Hk, D)), or with `cu` (n_seq + 1 first rows,
 * ascending from 0) S packed rows in all. Token i of n of sequence b gets position lengths[b] - n + i: `lengths`
 * count the new tokens. With tables (rows of at least D/2 by position, fp32 or `dtype`) keys are rotated on the
 * way as by trx_rope_fwd with fp32 tables, and with q (.., Hq, D) queries into q_out. A token whose position is
 * negative, behind the tables or on no page is not written and its rows of q_out are 0; so are q_out's rows behind
 * the last sequence. Two tokens at one place leave either's values, or parts of both.
 * strides: (sequence, token, head) of q, k, v, q_out (packed: the first is not used), then the cache's.
 */
int trx_paged_append(const void* q_or_null, const void* k, const void* v, void* q_out, void* k_pages,
                     void* v_pages, float* k_scales_or_null, float* v_scales_or_null,
                     const int32_t* block_table, const int32_t* lengths, const int32_t* cu_or_null,
                     const void* cos_or_null, const void* sin_or_null, int64_t n_seq, int64_t S, int64_t Hq,
                     int64_t Hk, int64_t D, int64_t pages, int64_t page_size, int64_t width,
                     const int64_t strides[23], int64_t table_rows, int64_t table_row_stride, int table_dtype,
                     int dtype, void* stream);

/*
 * Read back: rows cu[b] .. cu[b + 1] - 1 of k_out and v_out (rows, Hk, D), contiguous, become the first of sequence
 * b's in the cache, as trx_attn_fwd_packed takes them. Rows behind the last sequence become 0 with `zero_rest`, else
 * stay. strides: the cache's.
 */
int trx_paged_gather(const void* k_pages, const void* v_pages, const float* k_scales_or_null,
                     const float* v_scales_or_null, const int32_t* block_table, const int32_t* cu, void* k_out,
                     void* v_out, int64_t n_seq, int64_t rows, int64_t Hk, int64_t D, int64_t pages,
                     int64_t page_size, int64_t width, const int64_t strides[11], int zero_rest, int dtype,
                     void* stream);

/*
 * Causal attention of the last Sq tokens of each sequence, q (B, Sq, Hq, D), over the lengths[b] keys of it in the
 * cache, theirs among them: query i stands at position lengths[b] - Sq + i and sees the keys up to there, with
 * window_left >= 0 only the last window_left + 1 of these. slopes: ALiBi. A query that sees nothing is 0, its
 * LSE -inf. For few rows (decoding, drafts): the time grows with every 16 of Sq * Hq / Hk.
 * strides: (batch, token, head) of q, out, then the cache's. `parts` is trx_attn_paged_bytes() of device memory,
 * 16-byte aligned, for this call alone; it holds nothing between calls. Workspace and status as for trx_attn_fwd.
 */
int trx_attn_fwd_paged(const void* q, const void* k_pages, const void* v_pages, const float* k_scales_or_null,
                       const float* v_scales_or_null, void* out, float* lse_or_null,
                       const float* slopes_or_null, const int32_t* block_table, const int32_t* lengths,
                       int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D, int64_t pages,
                       int64_t page_size, int64_t width, const int64_t strides[17], float scale,
                       int64_t window_left, int dtype, void* parts_or_null, size_t parts_bytes,
                       void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of `parts` on the current device, 0 for none; keys: width * page_size. */
size_t trx_attn_paged_bytes(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D, int64_t keys,
                            int64_t window_left, int four_bits);

/*
 * Attach a word of pinned host memory to an attention workspace (NULL detaches it; the workspace
 * must have been zeroed before). From then on every launch on that workspace that gives up on a
 * bounded wait, or that finds such a failure recorded and skips its work, also writes the status
 * word there; a launch that works touches nothing. A host that reads the word before each call
 * needs no trx_attn_status copies. The caller keeps the word alive as long as it is attached, and
 * after a failure zeroes the device word first and this one when no launch queued before that is
 * left (each of them reports the failure again). One small launch on `stream`. Replaces nothing in
 * the reference.
 */
int trx_attn_mirror(void* workspace, unsigned int* host_word_or_null, void* stream);

/*
 * trx_attn_fwd for callers that cannot provide a workspace. No counterpart in the reference.
 *
 * Who needs it: hosts that pass pointers in but cannot create device memory when the call is
 * made — an inference-engine plugin whose memory plan is fixed when the engine is built and
 * whose execute hook must not allocate, or a process whose device memory is owned entirely by
 * a broker. This entry point performs no cudaMalloc / cudaFree and calls no allocating library
 * routine; the kernel's 256-byte scratch block lives in a static array inside the library
 * (256 bytes on every GPU that loads the library, kept until the process exits).
 *
 * Same arguments and results as trx_attn_fwd, minus the workspace, plus
 *   status_out_or_null: optional 4-byte destination (device or pinned host memory) that
 *   receives the kernel's status word in stream order; 0 means no bounded wait gave up.
 * Limit: the static block is 256 bytes, which is what the kernel needs for EVERY problem size
 * trx_attn_fwd accepts; if the library's own requirement ever exceeds the block the call
 * returns TRX_ERR_WORKSPACE and launches nothing.
 * Arguments are checked before the block is cleared, so an argument error enqueues nothing.
 * The one error that can follow the launch is TRX_ERR_CUDA from the 4-byte copy into
 * status_out_or_null; the attention output is valid all the same.
 * The first call on each device looks up the block's device address (with that device
 * current); make that first call outside of any stream capture.
 * All calls on a device share the one block, which still holds the previous call's contents:
 * the entry point zeroes it in stream order before each launch. Two calls whose work overlaps
 * on the GPU (different streams, or different host threads feeding different streams) race
 * on it; issue them on one stream or serialise them.
 */
int trx_attn_fwd_static_scratch(const void* q, const void* k, const void* v, void* out,
                                float* lse_or_null, const float* slopes_or_null, int64_t B,
                                int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hk, int64_t D,
                                const int64_t q_strides[3], const int64_t k_strides[3],
                                const int64_t v_strides[3], const int64_t o_strides[3],
                                float scale, int causal, int64_t window_left, int64_t window_right,
                                int dtype, unsigned int* status_out_or_null, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TRINIX_B200_H_ */
