/*
 * krsi_b200.h - C ABI of the B200 (sm_100a) kernels behind kernel-rsi's library ops.
 *
 * Every entry point takes plain device pointers, sizes and a cudaStream_t, launches
 * asynchronously on that stream, never synchronises, never allocates device memory and
 * returns a krsi_status code (0 = success).  Callers own all buffers; kernels that need
 * scratch memory take a caller-provided workspace whose size is reported by the matching
 * *_workspace_size() query.  Calls run on the CUDA context current to the calling thread,
 * and the stream must belong to that context.
 *
 * Each function names the reference interface it replaces (file:line inside the
 * kernel-rsi project).  Tensor layouts are the reference's:
 *   - rows are contiguous, row-major ("x2d" [rows, n], "u" [rows, 2F]);
 *   - qkv is [B*S, 3*H*D] with row stride `qkv_row_stride` elements and column layout
 *     [3][H][D]; out/out32 are [B*S, H*D] contiguous; lse and delta are [B*H, S];
 *   - pd is the per-head, per-distance bias [H, 2S-1] fp32:
 *     bias[h, i, j] = pd[h, j - i + S - 1].
 */
#ifndef KRSI_B200_H
#define KRSI_B200_H

#include <stddef.h>
#include <stdint.h>
#include <cuda_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes returned by every entry point. */
typedef enum {
  KRSI_OK = 0,
  KRSI_ERR_INVALID_ARGUMENT = 1, /* null pointer, bad size, stride or dtype combination   */
  KRSI_ERR_UNSUPPORTED = 2,      /* valid for the reference, not implemented here         */
  KRSI_ERR_MISALIGNED = 3,       /* pointer/stride alignment required by TMA or vector IO */
  KRSI_ERR_WORKSPACE = 4,        /* workspace pointer null or smaller than required       */
  KRSI_ERR_CUDA = 5,             /* a CUDA runtime/driver call failed (launch, attribute) */
  KRSI_ERR_DEVICE_TIMEOUT = 6    /* a bounded device-side wait gave up (see status read)  */
} krsi_status;

/* Element types accepted by the entry points. */
typedef enum { KRSI_F32 = 0, KRSI_BF16 = 1, KRSI_F16 = 2 } krsi_dtype;

/* Human-readable text for a krsi_status value. */
const char* krsi_error_string(int status);

/* ABI version: major*10000 + minor*100 + patch. */
int krsi_abi_version(void);

/* Reads (and optionally clears) the device-side watchdog word of the current device:
 * 0 when no bounded wait ever gave up, else a KRSI_ERR_DEVICE_TIMEOUT code with the
 * waiting role in bits 8..15.  Synchronises the current device; not for hot paths. */
int krsi_device_status(int* status_out, int clear);

/* ---------------------------------------------------------------- RMSNorm
 * y = w * (x * rstd).to(w.dtype), rstd = 1/sqrt(mean(x^2) + eps), per row.
 * Replaces library/rmsnorm.py:54-59 (_fwd -> _rms_fwd, rmsnorm.py:22-31).
 * x, y: [rows, n] of x_dtype; w: [n] of w_dtype; rstd: [rows] fp32. */
int krsi_rmsnorm_fwd(const void* x, const void* w, void* y, float* rstd,
                     int64_t rows, int64_t n, float eps,
                     int x_dtype, int w_dtype, cudaStream_t stream);

/* Bytes of workspace krsi_rmsnorm_bwd needs (the per-block dw partial sums). */
int krsi_rmsnorm_bwd_workspace_size(int64_t rows, int64_t n, size_t* bytes);

/* dx = r*dn - x*r^3*mean(dn*x) with dn = (g*w) rounded to the promoted input type;
 * dw = sum over rows of g * (x*r).to(w.dtype), reduced deterministically in two stages.
 * Replaces library/rmsnorm.py:62-68 (_bwd -> _rms_bwd, rmsnorm.py:34-51, then dwp.sum(0) at :68).
 * g, x, dx: [rows, n] of x_dtype; w, dw: [n] of w_dtype; rstd: [rows] fp32. */
int krsi_rmsnorm_bwd(const void* g, const void* x, const void* w, const float* rstd,
                     void* dx, void* dw, void* workspace, size_t workspace_bytes,
                     int64_t rows, int64_t n, int x_dtype, int w_dtype, cudaStream_t stream);

/* The same backward with a second gradient of x added: dx = (the backward above) + gadd, rounded
 * once.  For a pre-norm residual block, where x also feeds the residual branch and autograd would
 * otherwise add the two gradients of x in a separate pass (read both, write the sum).  No
 * counterpart in the reference (its backward returns dx alone, rmsnorm.py:62-68).
 * gadd: [rows, n] of x_dtype (16-byte aligned when n is a multiple of the vector width). */
int krsi_rmsnorm_bwd_add(const void* g, const void* x, const void* w, const float* rstd, const void* gadd,
                         void* dx, void* dw, void* workspace, size_t workspace_bytes,
                         int64_t rows, int64_t n, int x_dtype, int w_dtype, cudaStream_t stream);

/* The same backward for callers that cannot allocate device memory (a host that owns all device
 * memory, or a loop that must not stall on cudaMalloc): the dw partial sums live in a fixed
 * device array inside this library (4 MiB per GPU that loads it, kept until the process exits)
 * instead of a caller workspace.  No counterpart in the reference (its backward allocates
 * through torch, rmsnorm.py:66).
 * Limit: (dw partial rows) x n <= 1,048,576 floats.  The partial-row count is
 * min(ceil(rows / 8), 296) when one warp handles a row (rows of up to 2048 fp32 or 4096
 * 16-bit elements, 16-byte aligned) and min(rows, 296) otherwise; for example rows = 2048,
 * n = 1152 uses 256 x 1152.  Larger problems return KRSI_ERR_UNSUPPORTED.
 * Every call looks up the array's address (cudaGetSymbolAddress) in the current context, so a
 * device reset never leaves a stale pointer; the first call on a device also loads the module,
 * so make it before any stream capture.  All calls share the array:
 * calls whose kernels overlap on the GPU (different streams, same device) race and corrupt dw.
 * Allocates nothing: no cudaMalloc, cudaFree or allocating library call. */
int krsi_rmsnorm_bwd_noalloc(const void* g, const void* x, const void* w, const float* rstd,
                             void* dx, void* dw, int64_t rows, int64_t n, int x_dtype, int w_dtype,
                             cudaStream_t stream);

/* ---------------------------------------------------------------- GEGLU
 * out = gelu_tanh(u[:, :F]).to(dtype) * u[:, F:].
 * Replaces library/geglu.py:55-61 (_fwd -> _geglu_fwd, geglu.py:27-35).
 * u: [rows, 2F]; out: [rows, F]; both of `dtype`. */
int krsi_geglu_fwd(const void* u, void* out, int64_t rows, int64_t F, int dtype,
                   cudaStream_t stream);

/* du = [d(gate) | d(value)] in one [rows, 2F] tensor.
 * Replaces library/geglu.py:64-68 (_bwd -> _geglu_bwd, geglu.py:38-52).
 * g: [rows, F]; u, du: [rows, 2F]; all of `dtype`. */
int krsi_geglu_bwd(const void* g, const void* u, void* du, int64_t rows, int64_t F,
                   int dtype, cudaStream_t stream);

/* The gate|value projection with GEGLU in its epilogue (tcgen05 GEMM, fp32 accumulate):
 *   u = x @ w^T (rounded to dtype), out = gelu_tanh(u[:, :F]).to(dtype) * u[:, F:]
 * with krsi_geglu_fwd's arithmetic on the rounded u, so out equals krsi_geglu_fwd(u) bit for bit.
 * Replaces the T5 feed-forward's `geglu(h @ wi.T)`: the projection followed by
 * library/geglu.py:104-108 (geglu -> _fwd, geglu.py:55-61 -> _geglu_fwd, geglu.py:27-35).
 * x: [rows, K]; w: [2F, K] (rows [0, F) gate, [F, 2F) value); u: [rows, 2F]; out: [rows, F];
 * all of `dtype` (BF16 or F16), contiguous, 16-byte aligned; K and F multiples of 8. */
int krsi_linear_geglu_fwd(const void* x, const void* w, void* u, void* out, int64_t rows,
                          int64_t K, int64_t F, int dtype, cudaStream_t stream);

/* The down projection's input gradient with GEGLU's backward in its epilogue (tcgen05 GEMM):
 *   g = dy @ w (fp32 accumulate, rounded to dtype; never written), du = geglu_bwd(g, u)
 * with krsi_geglu_bwd's arithmetic, so du equals krsi_geglu_bwd(g, u) bit for bit for the rounded g.
 * Replaces the backward of the T5 feed-forward's `geglu(h @ wi.T) @ wo.T` from the down projection's
 * input gradient through GEGLU: `dy @ wo` followed by library/geglu.py:64-68 (_bwd -> _geglu_bwd,
 * geglu.py:38-52).
 * dy: [rows, K]; w: [K, F] (the down projection's weight, nn.Linear layout); u: [rows, 2F] (the
 * gate|value projection's output); du: [rows, 2F]; all of `dtype` (BF16 or F16), contiguous,
 * 16-byte aligned; K and F multiples of 8. */
int krsi_linear_geglu_bwd(const void* dy, const void* w, const void* u, void* du, int64_t rows,
                          int64_t K, int64_t F, int dtype, cudaStream_t stream);

/* ---------------------------------------------------------------- relpos attention
 * Flash attention with an additive Toeplitz bias, non-causal:
 *   s2[i,j] = (q_i . k_j * scale + pd[h, j-i+S-1]) * log2(e),  p = softmax over j,
 *   out = p @ v  (bf16 or f16, [B*S, H*D]),  out32 = same in fp32,
 *   lse[b*H+h, i] = max_j s2 + log2(sum_j exp2(s2 - max))   (log2 domain).
 * Replaces library/relpos_attention.py:132-140 (_forward -> _fwd, relpos_attention.py:26-59).
 * D must be a multiple of 8 and <= 128; qkv_row_stride a multiple of 8; dtype BF16 or F16. */
int krsi_relpos_attn_fwd(const void* qkv, int64_t qkv_row_stride, const float* pd,
                         void* out, float* out32, float* lse,
                         int64_t B, int64_t S, int64_t H, int64_t D, float scale,
                         int dtype, cudaStream_t stream);

/* Bytes of workspace krsi_relpos_attn_bwd needs (delta, fp32 dQ accumulator,
 * per-tile dBias diagonal partials). */
int krsi_relpos_attn_bwd_workspace_size(int64_t B, int64_t S, int64_t H, int64_t D,
                                        size_t* bytes);

/* Gradients of the forward above for upstream gradient dout [B*S, H*D] (contiguous):
 *   dqkv [B*S, 3*H*D] (row stride dqkv_row_stride, same [3][H][D] column layout),
 *   dpd  [H, 2S-1] fp32 = sum over batch of the diagonal sums of dS (unscaled).
 * delta = rowsum(dout * out32) is computed from the fp32 copy of O.
 * Replaces library/relpos_attention.py:143-157 (_backward_impl -> _bwd_dkdv :62-94,
 * _bwd_dq :97-126 and the torch diagonal reduction :154-156). */
int krsi_relpos_attn_bwd(const void* dout, const void* qkv, int64_t qkv_row_stride,
                         const float* pd, const float* out32, const float* lse,
                         void* dqkv, int64_t dqkv_row_stride, float* dpd,
                         void* workspace, size_t workspace_bytes,
                         int64_t B, int64_t S, int64_t H, int64_t D, float scale,
                         int dtype, cudaStream_t stream);

/* ---------------------------------------------------------------- T5 bucketed relative position
 * The step either side of the attention op in a T5 model (its relative_attention_bias table).
 * T5's bucket of a distance rel = key - query (HF transformers T5Attention._relative_position_bucket,
 * models/t5/modeling_t5.py): with n = num_buckets / 2 if bidirectional (rel > 0 adds n) else
 * num_buckets, e = n / 2 and a = |rel| (bidirectional) or max(-rel, 0): bucket offset a for a < e,
 * else e + trunc(log(a / e) / log(max_distance / e) * (n - e)), capped at n - 1.
 * The reference's attention op takes the bias per distance (pd [H, 2S-1], relpos_attention.py:5);
 * the reference leaves the table -> pd step and its gradient to torch (an embedding lookup, and
 * an S x S scatter-add in its backward, LESSONS.md:35). */

/* Bucket of one distance (host-side, no device work): the map the kernels below use. */
int krsi_t5_bucket(int num_buckets, int max_distance, int bidirectional, int64_t rel, int* bucket);

/* pd[h, t] = table[bucket(t - (S - 1)), h] for t in [0, 2S - 1).
 * table: [num_buckets, H] of table_dtype (F32, BF16, F16); pd: [H, 2S - 1] fp32. */
int krsi_t5_bias_fwd(const void* table, float* pd, int64_t S, int64_t H, int num_buckets, int max_distance,
                     int bidirectional, int table_dtype, cudaStream_t stream);

/* dtable[k, h] = sum of dpd[h, t] over the distances t - (S - 1) in bucket k (a segmented sum in a
 * fixed order: deterministic), rounded to table_dtype.  dpd: [H, 2S - 1] fp32. */
int krsi_t5_bias_bwd(const float* dpd, void* dtable, int64_t S, int64_t H, int num_buckets, int max_distance,
                     int bidirectional, int table_dtype, cudaStream_t stream);

/* ---------------------------------------------------------------- embedding
 * out[i] = scale * table[tokens[i]] and the table's gradient.  The reference has no embedding op (its
 * models leave the lookup to torch).
 * tokens: [n] of token_bits 32 or 64 (int32/int64); table, dtable: [V, d]; out, g: [n, d]; all but the
 * tokens of `dtype`, contiguous.  A token outside [0, V) gives a row of NaN and no gradient. */
int krsi_embedding_fwd(const void* tokens, int token_bits, const void* table, void* out, int64_t n,
                       int64_t V, int64_t d, float scale, int dtype, cudaStream_t stream);

/* Bytes of workspace krsi_embedding_bwd needs (the sorted positions and the partial rows of tokens
 * that occur often). */
int krsi_embedding_bwd_workspace_size(int64_t n, int64_t V, int64_t d, size_t* bytes);

/* dtable[v] = scale * sum of g[i] over the i with tokens[i] = v, summed in fp32 in a fixed order over
 * the sorted positions (deterministic, no atomics) and rounded once; every row of dtable is written.
 * padding_idx: a token whose row gets no gradient, or -1.  workspace: 16-byte aligned. */
int krsi_embedding_bwd(const void* tokens, int token_bits, const void* g, void* dtable, void* workspace,
                       size_t workspace_bytes, int64_t n, int64_t V, int64_t d, float scale,
                       int64_t padding_idx, int dtype, cudaStream_t stream);

/* ---------------------------------------------------------------- GEGLU with an 8-bit checkpoint
 * krsi_geglu_fwd/bwd with u kept for the backward in 8 bits.  No counterpart in the reference (its
 * backward reads u in full, geglu.py:64-68).
 * The checkpoint: q [rows, 2F] int8 and exponents [rows, ceil(F / 32), 2] uint8 (gate, value; 2-byte
 * aligned); in a
 * group of 32 columns of a half-row u is kept as q * 2^(e - 127), with 2^(e - 127) = 2^-6 of the power
 * of two at or below the group's largest magnitude (2^-126 at least) and q rounded to nearest even
 * within [-127, 127].  e = 255 marks a group with a value that is not finite: it reads back as NaN.
 * out = gelu_tanh(u[:, :F]) * u[:, F:] from u itself, in fp32, rounded once (krsi_geglu_fwd rounds
 * gelu_tanh to dtype before the product).  q and exponents both null: no checkpoint, out alone. */
int krsi_geglu_q8_fwd(const void* u, void* out, void* q, void* exponents, int64_t rows, int64_t F, int dtype,
                      cudaStream_t stream);

/* du = [d(gate) | d(value)] of GEGLU at the checkpoint's values, for g [rows, F]; and, where out is not
 * null, out [rows, F] = GEGLU of those values (an operand of the down projection's weight gradient). */
int krsi_geglu_q8_bwd(const void* g, const void* q, const void* exponents, void* du, void* out, int64_t rows,
                      int64_t F, int dtype, cudaStream_t stream);

/* ---------------------------------------------------------------- vocabulary cross entropy
 * Softmax cross entropy of a projection onto the vocabulary, and both gradients, without the [N, V]
 * logits in memory.  The reference has no loss op.
 *   l = scale * x @ w^T, lse_i = log sum_v exp(l[i, v]),
 *   loss_i = lse_i - l[i, t_i] + z_loss * lse_i^2, 0 for an ignored row.
 * x, dx: [N, K]; w, dw: [V, K]; `dtype` BF16 or F16, contiguous, 16-byte aligned; K a multiple of 8.
 * targets: [N] of target_bits 32 or 64; a row whose target is ignore_index has loss and gradients of
 * zero, whatever its x holds; a target outside [0, V) that is not ignore_index makes the loss and the
 * gradients NaN.  workspace: 256-byte aligned.  Needs clusters of two CTAs (KRSI_ERR_UNSUPPORTED where
 * the device has none). */

/* Bytes of workspace: mode 0 krsi_linear_ce_fwd without gradients, 1 with, 2 krsi_linear_ce_grad; 1 and 2 less what
 * one gradient takes with KRSI_CE_NO_DX or KRSI_CE_NO_DW added, for calls where that pointer is null.
 * A call works on chunks of rows: R rows, of at least 256.  In bytes, each part rounded up to 256:
 *   always     16 N; mode 0 and 1: 16 R ceil(V / 256), at most 2^28 for the loss alone (or 256 rows')
 *   gradients  20 N + R (128 ceil(V / 64) + 2 K), R so that the first product is at most 2^29 (or 256 rows')
 *   dx         4 R K for each share of the vocabulary that its sums are cut into (none where R is large)
 *   dw         with more than 512 rows the sorted targets, about 4 V + 8 N + N K / 2; mode 2: 4 K for each
 *              row of w, or in one chunk for each row of x where those are fewer and w's take over 32 MB */
#define KRSI_CE_NO_DX 4
#define KRSI_CE_NO_DW 8
int krsi_linear_ce_workspace_size(int64_t N, int64_t V, int64_t K, int mode, size_t* bytes);

/* loss: [N] fp32.  total, weight: one float each, or both null: the sum of the losses (mean: divided by
 * the number of rows that are not ignored, at least 1), and the weight of one row in it (1, or one over
 * that number).
 * stats: [N, 2] fp32 for krsi_linear_ce_grad (8-byte aligned), or null.
 * dx, dw: null, or fp32 gradients of the sum of the losses without the factor `scale`, for
 * krsi_linear_ce_finish: the logits are computed once for loss and gradients. */
int krsi_linear_ce_fwd(const void* x, const void* w, const void* targets, int target_bits, float* loss,
                       float* total, float* weight, float* stats, float* dx, float* dw, void* workspace,
                       size_t workspace_bytes, int64_t N, int64_t V, int64_t K, float scale, int64_t ignore_index,
                       float z_loss, int mean, int dtype, cudaStream_t stream);

/* Gradients for the upstream gradient g of each row's loss (fp32, stride 1, or 0: one for all rows), times
 * *weight where that is not null, from the stats of krsi_linear_ce_fwd on the same operands (the logits
 * are computed again).  dx, dw: of `dtype`, one of them may be null. */
int krsi_linear_ce_grad(const void* x, const void* w, const void* targets, int target_bits, const float* g,
                        int64_t g_stride, const float* weight, const float* stats, void* dx, void* dw,
                        void* workspace, size_t workspace_bytes, int64_t N, int64_t V, int64_t K, float scale,
                        int64_t ignore_index, float z_loss, int dtype, cudaStream_t stream);

/* out = scale * *g * *weight * grad, rounded once (g, weight: device scalars or null); n a multiple of 8. */
int krsi_linear_ce_finish(const float* grad, const float* g, const float* weight, void* out, int64_t n,
                          float scale, int dtype, cudaStream_t stream);

/* ---------------------------------------------------------------- residual addition and RMSNorm
 * z = (x + res) rounded to x_dtype, rstd = 1 / sqrt(mean(z^2) + eps), y = w * z * rstd in fp32, rounded once
 * (krsi_rmsnorm_fwd rounds z * rstd first).  The reference has no such op (its models add, then call
 * library/rmsnorm.py:22-31).
 * x, res, z, y: [rows, n] of x_dtype; w: [n] of w_dtype; contiguous; dtypes as krsi_rmsnorm_fwd's; n up to 16384
 * (32768 for 16-bit x with rows of whole 16 bytes at 16-byte aligned pointers).
 * res null: z is x, and is not written. */
int krsi_add_rmsnorm_fwd(const void* x, const void* res, const void* w, void* z, void* y, float* rstd,
                         int64_t rows, int64_t n, float eps, int x_dtype, int w_dtype, cudaStream_t stream);

int krsi_add_rmsnorm_bwd_workspace_size(int64_t rows, int64_t n, size_t* bytes);

/* dz = gy * w * rstd - z * rstd^3 * mean(gy * w * z) + gz, the gradient of x and of res, and dw = sum of gy * z * rstd
 * over the rows, both in fp32 with one rounding (krsi_rmsnorm_bwd_add rounds gy * w and z * rstd on the way); dw's
 * sum has a fixed order.  gz null: none. */
int krsi_add_rmsnorm_bwd(const void* gy, const void* gz, const void* z, const void* w, const float* rstd, void* dz,
                         void* dw, void* workspace, size_t workspace_bytes, int64_t rows, int64_t n, int x_dtype,
                         int w_dtype, cudaStream_t stream);

/* The same with y in 8 bits: q [rows, n] e4m3, row i at q + i * q_stride bytes, and scale [rows] fp32;
 * y = q * scale, q = e4m3(z * w * (448 / m)) and scale = m * rstd / 448 for the row's largest |z * w| m.
 * A row with a value that is not finite has a scale that is not finite. */
int krsi_add_rmsnorm_q8_fwd(const void* x, const void* res, const void* w, void* z, void* q, int64_t q_stride,
                            float* scale, int64_t rows, int64_t n, float eps, int x_dtype, int w_dtype,
                            cudaStream_t stream);

/* Rows in 8 bits: q = e4m3(x * (448 / m)), scale = m / 448 for the row's largest |x| m. */
int krsi_quantise_rows(const void* x, void* q, int64_t q_stride, float* scale, int64_t rows, int64_t n, int x_dtype,
                       cudaStream_t stream);

/* ---------------------------------------------------------------- product of rows and a weight in 8 bits
 * out[i, j] = (sum over k of q[i, k] * wq[j, k]) * scale[i] * wscale[j], summed in fp32, rounded once.
 * q: rows of K e4m3, q_stride bytes apart; wq: M rows of K e4m3, w_stride bytes apart (both strides multiples of
 * 16, both bases 16-byte aligned); out: [rows, M] of out_dtype, contiguous.  No counterpart in the reference. */
int krsi_linear_q8(const void* q, int64_t q_stride, const float* scale, const void* wq, int64_t w_stride,
                   const float* wscale, void* out, int64_t rows, int64_t K, int64_t M, int out_dtype,
                   cudaStream_t stream);

/* ---------------------------------------------------------------- AdamW over many tensors
 * One step for every tensor of the list, in place; no counterpart in the reference (its models leave the
 * optimizer to torch).  With g' = g * min(1, max_norm / (|all g| + 1e-6)), or g where max_norm is 0:
 *   t = t + 1,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
 *   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
 * A norm that is not finite leaves everything as it is, the step included. */

/* Added to state_bits 8: m's codes are rounded up or down at random, right on average, as those of sqrt(v) always are.
 * Without it m's codes are the nearest ones, which is right for one step and not for a run of them: m stops wherever
 * (1 - b1) |g' - m| is below half a code. */
#define KRSI_ADAMW_RANDOM_M 256

typedef struct {
  void* p;            /* [n] of p_dtype */
  const void* g;      /* [n] of g_dtype: p_dtype or F32 */
  void* m;            /* state_bits 32: fp32 m and v; 8, alone or + KRSI_ADAMW_RANDOM_M: e4m3 codes of m and of sqrt(v) */
  void* v;
  float* master;      /* fp32 copy of a 16-bit p that is updated in its place (p: its rounding), or null */
  uint8_t* exponents; /* 8-bit states: [ceil(n / 256), 2]: a group of 256 codes stands for code * 2^(e - 127),
                         e of m and of sqrt(v); 255 marks a group that is not finite (it reads back as NaN).
                         2-byte aligned */
  int64_t n;
  int p_dtype, g_dtype, state_bits, reserved;
} krsi_adamw_tensor;

int krsi_adamw_workspace_size(int64_t count, size_t* bytes);

/* tensors: host memory, read during the call only; no two of them may overlap.  step: device, the steps taken so
 * far.  lr_dev: a device float that is read in place of lr, or null.  norm_out: device, the norm of all gradients
 * (max_norm > 0 only).  workspace: 16-byte aligned. */
int krsi_adamw_step(const krsi_adamw_tensor* tensors, int64_t count, int64_t* step, const float* lr_dev, double lr,
                    double beta1, double beta2, double eps, double weight_decay, double max_norm, float* norm_out,
                    void* workspace, size_t workspace_bytes, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KRSI_B200_H */
