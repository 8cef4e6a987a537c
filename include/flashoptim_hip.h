/*
 * flashoptim_hip.h -- C ABI of libflashoptim_hip.so, the gfx950 (MI355X) implementation of FlashOptim's
 * fused optimizer-step hot path.
 *
 * Every entry point takes raw device pointers, sizes, fp32 scalars and a HIP stream (as void*); none takes
 * a torch type, allocates tensor memory or synchronises with the host.  All work is enqueued on `stream`
 * and mutates the caller's buffers in place, exactly as the reference's Triton launch wrappers do.
 * Return value: 0 on success, otherwise a negative FO_ERR_* code or a positive hipError_t; the text of the
 * last failure on the calling thread is available from fo_last_error().  Nothing throws across the ABI.
 *
 * "ref:" cites /root/reference/flashoptim/optimizers.py, the interface each symbol replaces.
 *
 * Layout contract shared by all entry points (ref:2476-2484, 1625-1646):
 *   - tensors are flat and contiguous; element i of the parameter pairs with element i of grad, ecc, codes;
 *   - a quantisation group is 32 consecutive elements counted from element 0 of the tensor; scales are
 *     fp16, one per group, ceil(n/32) entries; a short last group is scaled by its own absmax;
 *   - first-moment codes are int8 (softsign companding), second-moment codes uint8 (of sqrt(v));
 *   - ECC is int8 (24-bit master) or int16 (32-bit master), absent for fp32 parameters.
 */
#ifndef FLASHOPTIM_HIP_H
#define FLASHOPTIM_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* parameter / gradient element type (ref:60-64 _TORCH_DTYPE_TO_TRITON_DTYPE) */
enum fo_dtype { FO_F32 = 0, FO_BF16 = 1, FO_F16 = 2 };

enum fo_error {
    FO_OK = 0,
    FO_ERR_INVALID_ARGUMENT = -1, /* bad enum, null pointer, negative size, misaligned scale pointer ... */
    FO_ERR_UNSUPPORTED = -2,      /* e.g. ECC requested for an fp32 parameter */
    FO_ERR_NO_DEVICE = -3
};

/* Library / device identification. */
int fo_version(void);                    /* 100*major + minor */
const char *fo_last_error(void);         /* thread-local, never NULL */
int fo_device_compute_units(int device); /* multiprocessor count, <0 on error (ref:2976-2980 _get_sm_count) */

/*
 * Fused Adam / AdamW step on one tensor.  Replaces _fused_adam_step + _triton_adam_kernel
 * (ref:2203-2251, 2255-2438).
 *   mom, var        : quantized != 0 -> int8 / uint8 codes; else tensors of the parameter dtype
 *   mom_scales,
 *   var_scales      : fp16[ceil(n/32)] when quantized, ignored otherwise (may be NULL)
 *   param, grad     : `dtype` elements; grad is read only
 *   ecc             : int8 (ecc_bytes 1) / int16 (ecc_bytes 2) / NULL (ecc_bytes 0)
 *   weight_decay    : what the reference launcher passes: already multiplied by lr (or lr/initial_lr) for the
 *                     decoupled optimizers, the raw L2 coefficient otherwise (ref:1894-1898)
 *   step            : 1-based step count used for bias correction (ref:2368-2369)
 */
int fo_adam_step(void *mom, void *mom_scales, void *var, void *var_scales, void *param, const void *grad,
                 void *ecc, int64_t n, int dtype, int ecc_bytes, int quantized, float lr, float beta1,
                 float beta2, float eps, float weight_decay, int decoupled, int step, void *stream);

/*
 * Fused SGD / SGDW / Nesterov / Lion step on one tensor.  Replaces _fused_momentum_step +
 * _triton_momentum_kernel (ref:1535-1579, 1586-1719).  Lion: mom_coef = beta2, update_coef = beta1,
 * do_lion = 1 (ref:1313-1317); SGD: mom_coef = momentum, update_coef = 1 - dampening (ref:1432-1433).
 */
int fo_momentum_step(void *mom, void *mom_scales, void *param, const void *grad, void *ecc, int64_t n,
                     int dtype, int ecc_bytes, int quantized, float lr, float mom_coef, float update_coef,
                     float weight_decay, int decoupled, int nesterov, int do_lion, void *stream);

/*
 * Momentum-free SGD step (no state tensor).  Replaces the eager branch the reference takes when
 * momentum == 0 (ref:1447-1465): both decays are skipped when weight_decay == 0.
 */
int fo_sgd_plain_step(void *param, const void *grad, void *ecc, int64_t n, int dtype, int ecc_bytes, float lr,
                      float weight_decay, int decoupled, void *stream);

/*
 * Multi-tensor launch: one grid over many tensors of ragged sizes (no counterpart in the reference, which
 * launches once per tensor from FlashOptimizer.step, ref:770-785; results are bit-identical to calling the
 * single-tensor entry point on every tensor).
 *
 * `descs` is a DEVICE array of n_tensors descriptors; `chunks` is a DEVICE array of n_chunks work items
 * produced by fo_build_chunks (host) and copied by the caller.  All tensors of one call share dtype,
 * ecc_bytes, quantized and the scalar hyper-parameters (callers bucket by those).
 */
typedef struct fo_tensor_desc {
    void *param;
    const void *grad;
    void *ecc;        /* NULL when ecc_bytes == 0 */
    void *mom;        /* first-moment state (codes or plain values) */
    void *mom_scales; /* NULL when not quantized */
    void *var;        /* Adam only */
    void *var_scales; /* Adam only, NULL when not quantized */
    int64_t n;        /* elements in this tensor */
} fo_tensor_desc;

typedef struct fo_chunk {
    int32_t tensor;     /* index into descs */
    int32_t first_tile; /* first 4096-element tile of the tensor covered by this chunk */
    int32_t n_tiles;    /* tiles covered (>= 1) */
    int32_t reserved;
} fo_chunk;

#ifndef FO_TILE_ELEMS
#define FO_TILE_ELEMS 4096
#endif

/* Host helper: number of chunks fo_build_chunks will emit for these tensor lengths (0-length tensors emit
 * none).  tiles_per_chunk <= 0 selects the library default. */
int64_t fo_count_chunks(const int64_t *numels, int64_t n_tensors, int tiles_per_chunk);
/* Host helper: fills `out` (host memory, capacity >= fo_count_chunks) and returns the count, <0 on error. */
int64_t fo_build_chunks(const int64_t *numels, int64_t n_tensors, int tiles_per_chunk, fo_chunk *out,
                        int64_t capacity);

int fo_multi_adam_step(const fo_tensor_desc *descs, int64_t n_tensors, const fo_chunk *chunks, int64_t n_chunks,
                       int dtype, int ecc_bytes, int quantized, float lr, float beta1, float beta2, float eps,
                       float weight_decay, int decoupled, int step, void *stream);

int fo_multi_momentum_step(const fo_tensor_desc *descs, int64_t n_tensors, const fo_chunk *chunks,
                           int64_t n_chunks, int dtype, int ecc_bytes, int quantized, float lr, float mom_coef,
                           float update_coef, float weight_decay, int decoupled, int nesterov, int do_lion,
                           void *stream);

/*
 * fo_multi_adam_step for callers that cannot allocate device memory or copy tables to it (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  It has no counterpart in the reference.
 * The caller passes the descriptors as a HOST array; the library keeps the descriptor and chunk tables in a static
 * device array of its own (FO_STATIC_MAX_TENSORS descriptors + FO_STATIC_MAX_CHUNKS chunk entries, 1.06 MiB per
 * device, held until the process ends), fills them with small kernels whose arguments carry the descriptors, and
 * launches the same step kernel.  It calls no hipMalloc / hipFree / hipMemcpy.  Lists with more than
 * FO_STATIC_MAX_TENSORS tensors are refused; lists with more than FO_STATIC_MAX_CHUNKS tiles are covered with
 * several 4096-element tiles per work item.  Results are bit-identical to fo_multi_adam_step.  All calls on one
 * device share the one array: calls that overlap in time on a device (different streams or threads) race.
 * The first call on a device, and the first call of each kernel variant (dtype, ecc_bytes, quantized, decoupled)
 * there, takes the array's address and plans the kernel's residency through host API calls that must not run while
 * the stream is capturing: make one eager call per variant before capturing.  After that a call enqueues kernel
 * launches only.  There is no `_exact` twin of this entry point: it runs what fo_multi_adam_step runs.
 */
#define FO_STATIC_MAX_TENSORS 1024
#define FO_STATIC_MAX_CHUNKS 65536
int fo_multi_adam_step_static(const fo_tensor_desc *host_descs, int64_t n_tensors, int dtype, int ecc_bytes,
                              int quantized, float lr, float beta1, float beta2, float eps, float weight_decay,
                              int decoupled, int step, void *stream);

/*
 * fo_adam_step / fo_multi_adam_step with the update evaluated operation by operation as the reference writes it,
 *     p -= (lr * (m / bc1)) / (sqrt(v / bc2) + eps)          (ref:2368-2375)
 * with correctly rounded quotients and roots, on every element and for every parameter dtype: every output bit
 * then equals an IEEE evaluation of the reference's formulas.
 * The plain entry points already do this wherever nothing else meets one unit of master precision: fp32
 * parameters, 2-byte parameters with a 2-byte ECC (32-bit masters), fp16 parameters with a 1-byte ECC.  For bf16
 * parameters with a 1-byte ECC (24-bit masters) and 2-byte parameters without ECC they fold the bias corrections
 * and the learning rate into two constants (one reciprocal per element) and redo operation by operation only the
 * elements whose update all but cancels the weight; moment codes and scales are then still bit-identical and
 * every master weight lies within one unit of master precision, but the correction code may differ by one step.
 * Same arguments and errors as the plain entry points.  The reference has one kernel and no such choice; these
 * are for callers who want every bit.
 */
int fo_adam_step_exact(void *mom, void *mom_scales, void *var, void *var_scales, void *param, const void *grad,
                       void *ecc, int64_t n, int dtype, int ecc_bytes, int quantized, float lr, float beta1,
                       float beta2, float eps, float weight_decay, int decoupled, int step, void *stream);
int fo_multi_adam_step_exact(const fo_tensor_desc *descs, int64_t n_tensors, const fo_chunk *chunks,
                             int64_t n_chunks, int dtype, int ecc_bytes, int quantized, float lr, float beta1,
                             float beta2, float eps, float weight_decay, int decoupled, int step, void *stream);

/* Momentum-free SGD over many tensors: the multi-tensor form of fo_sgd_plain_step (descs use param, grad, ecc, n). */
int fo_multi_sgd_plain_step(const fo_tensor_desc *descs, int64_t n_tensors, const fo_chunk *chunks,
                            int64_t n_chunks, int dtype, int ecc_bytes, float lr, float weight_decay,
                            int decoupled, void *stream);

/*
 * Largest magnitude of every tensor of a list in one launch.  Replaces the per-tensor
 * tensor.abs().max().item() behind check_numerics / recompute_param_stats (ref:656-673), which costs one device
 * synchronisation per tensor.  descs use `param` (the data, `dtype` elements) and `n`; `out` is fp32[n_tensors],
 * zeroed by the caller; out[i] receives max |x| of tensor i (NaN if it holds a NaN).  Chunks from
 * fo_build_chunks with any tiles_per_chunk (larger chunks mean fewer atomic merges).
 */
int fo_multi_absmax(const fo_tensor_desc *descs, int64_t n_tensors, const fo_chunk *chunks, int64_t n_chunks,
                    int dtype, float *out, void *stream);

/*
 * Standalone group codec.  Replaces quantize / dequantize and their kernels (ref:2446-2538, 2541-2676).
 *   x            : `x_dtype` elements
 *   codes        : int8 when is_signed, uint8 otherwise
 *   scales       : fp16[ceil(n/32)]
 */
int fo_quantize(const void *x, int x_dtype, void *codes, void *scales, int64_t n, int is_signed, int do_sqrt,
                int softsign, void *stream);
int fo_dequantize(const void *codes, const void *scales, float *out, int64_t n, int is_signed, int do_sqrt,
                  int softsign, void *stream);

/*
 * Standalone ECC.  fo_ecc_join replaces reconstruct_fp32_param (ref:2835-2892, kernel 2779-2803);
 * fo_ecc_split replaces compute_ecc_bits (ref:2895-2970, kernel 2806-2832).  narrow_dtype is FO_BF16 or
 * FO_F16; ecc_bytes is 1 or 2.
 */
int fo_ecc_join(const void *narrow, int narrow_dtype, const void *ecc, int ecc_bytes, float *out, int64_t n,
                void *stream);
int fo_ecc_split(const float *x, const void *narrow, int narrow_dtype, void *ecc, int ecc_bytes, int64_t n,
                 void *stream);

/*
 * The conversions of a checkpoint over a list of tensors: what the reference runs as one kernel and one eager cast per
 * state of every parameter while it writes or reads a state_dict (ref:159-210, 797-927).  `jobs` is a HOST array: the jobs travel as kernel arguments, 64 to a
 * launch, so nothing is allocated, uploaded or synchronised, and the calls may be captured into a HIP graph.  Tensors
 * of different lengths share a launch; jobs of no elements are skipped.  All jobs of one call live on the
 * current device.
 */
typedef struct fo_convert_job {
    const void *src;
    const void *src2;
    void *dst;
    void *dst2;
    int64_t n;      /* elements */
    int32_t flags;  /* codec jobs: FO_CODEC_* */
    int32_t reserved;
} fo_convert_job;

enum fo_codec_flags { FO_CODEC_SIGNED = 1, FO_CODEC_SQRT = 2, FO_CODEC_SOFTSIGN = 4 };

/* src = values (x_dtype), dst = codes, dst2 = scales */
int fo_quantize_many(const fo_convert_job *jobs, int64_t n_jobs, int x_dtype, void *stream);
/* src = codes, src2 = scales, dst = values: fp32, or bf16 rounded to nearest even from the fp32 value */
int fo_dequantize_many(const fo_convert_job *jobs, int64_t n_jobs, int out_dtype, void *stream);
/* int8 correction codes as values of the parameter's type (bf16 or fp16), the form a checkpoint holds them in
 * (ref:900-927): src = int8, dst = `dtype` values; and back, truncated towards zero: src = `dtype` values, dst = int8 */
int fo_int8_widen_many(const fo_convert_job *jobs, int64_t n_jobs, int dtype, void *stream);
int fo_int8_narrow_many(const fo_convert_job *jobs, int64_t n_jobs, int dtype, void *stream);

/* fp32 master weights out of the parameters (ref:1035-1084): src = narrow_dtype values, src2 = their ecc, dst = fp32 */
int fo_ecc_join_many(const fo_convert_job *jobs, int64_t n_jobs, int narrow_dtype, int ecc_bytes, void *stream);
/* and into them (ref:1086-1147): src = fp32, dst = narrow_dtype values rounded to nearest even,
 * dst2 = their ecc, as fo_ecc_split gives it for src and dst */
int fo_ecc_narrow_many(const fo_convert_job *jobs, int64_t n_jobs, int narrow_dtype, int ecc_bytes, void *stream);

/*
 * Newton-Schulz orthogonalisation and the Muon optimizer step (no counterpart in the reference).  For a matrix G, with X its
 * orientation of fewer rows than columns:  X <- G / (|G|_F + eps), then `steps` times X <- a X + (b S + c S S) X, S = X X'.
 * `coefficients` (host memory) is {a, b, c}.
 */
#define FO_MATRIX_MOST_LINES 65536 /* rows and columns of one matrix */

/* `count` matrices of one shape; lr: the optimizer step's learning rate for them */
typedef struct fo_matrix_shape {
    int32_t rows, cols, count;
    float lr;
} fo_matrix_shape;

/* Bytes of device memory, aligned to 256, that the calls below need for these shapes; negative: FO_ERR_* */
int64_t fo_newton_schulz_workspace(const fo_matrix_shape *shapes, int64_t n_shapes);

/* `count` matrices of `dtype`, `stride` elements apart, rows `row_stride` apart, columns adjacent; result: bfloat16, contiguous.
 * The workspace is free again when the call's work on `stream` is done. */
int fo_newton_schulz(const void *x, int dtype, int64_t count, int64_t rows, int64_t cols, int64_t stride, int64_t row_stride,
                     void *result, int steps, const float *coefficients, float eps, void *workspace, int64_t workspace_bytes,
                     void *stream);

/*
 * One step over a list of matrices: m <- mu m + (1 - mu) g (codes and scales requantised, or `dtype` values), the update
 * (nesterov: (1 - mu) g + mu m, else m) through the iteration above, p <- p * keep - lr * update at master precision.
 *   matrices: device memory, those of shapes[0] first, then those of shapes[1] and so on (var, var_scales and n are not
 *   looked at); shapes: host memory
 */
int fo_muon_step(const fo_tensor_desc *matrices, const fo_matrix_shape *shapes, int64_t n_shapes, int dtype, int ecc_bytes,
                 int quantized, float keep, float momentum_coef, int nesterov, int steps, const float *coefficients, float eps,
                 void *workspace, int64_t workspace_bytes, void *stream);

/*
 * Microscaled 4-bit floating point (MXFP4, no counterpart in the reference).  A row of `cols` values is stored as
 * 64 * ceil(cols / 128) bytes of E2M1 codes, two to a byte, the first in the low half, and 4 * ceil(cols / 128) E8M0 scale
 * bytes, one per 32 values; zeros fill it up.  Scale: floor(log2(largest magnitude)) - 2, codes rounded to nearest even, magnitudes
 * above 6 become 6; a group with an infinity or a NaN has scale byte 255.  Codes are aligned to 16 bytes, scales of a product to 4.
 */

/* x: rows x cols of `dtype`, rows `row_stride` elements apart, columns adjacent.  codes, scales: of the rows; column_codes,
 * column_scales: of the transpose (cols rows of `rows` values).  Either pair may be NULL. */
int fo_mxfp4_quantize(const void *x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void *codes, void *scales,
                      void *column_codes, void *column_scales, void *stream);

/* out: rows x cols of `dtype`, contiguous */
int fo_mxfp4_dequantize(const void *codes, const void *scales, int64_t rows, int64_t cols, void *out, int dtype, void *stream);

/* out[i][j] = sum over `inner` values of a[i] * b[j], summed in fp32; out: rows x cols of `dtype`, contiguous */
int fo_mxfp4_product(const void *a, const void *a_scales, int64_t rows, const void *b, const void *b_scales, int64_t cols, int64_t inner,
                     void *out, int dtype, void *stream);

/* The same for up to FO_MXFP4_MOST_TOKENS rows that are not quantised yet.  Where fo_mxfp4_tokens_workspace is 0 one launch
 * quantises and multiplies them; else they are quantised into a workspace of so many bytes of device memory, aligned to 16. */
#define FO_MXFP4_MOST_TOKENS 64
int64_t fo_mxfp4_tokens_workspace(int64_t tokens, int64_t inner);
int fo_mxfp4_tokens(const void *x, int x_dtype, int64_t tokens, int64_t row_stride, const void *weight, const void *weight_scales,
                    int64_t cols, int64_t inner, void *out, int dtype, void *workspace, int64_t workspace_bytes, void *stream);

/*
 * A linear layer, y = x weight', its products in this format.  A form here is a matrix's codes followed by its scales,
 * fo_mxfp4_form_bytes(rows, cols) bytes of it, aligned to 16 bytes.
 * Forward: x is tokens x inner, weight outer x inner, out tokens x outer of x's type.  x_columns (inner x tokens) and
 * weight_columns (inner x outer), the forms of the transposes, are what the backward pass needs; either may be NULL.
 *   workspace: the forms of x and of weight.
 * Backward: dy is tokens x outer; dx = dy weight (tokens x inner) needs weight_columns, dw = dy' x (outer x inner) x_columns; either
 * may be left out (NULL).  workspace: the form of dy for dx, of its transpose for dw.
 */
int64_t fo_mxfp4_form_bytes(int64_t rows, int64_t cols);
int fo_mxfp4_linear_forward(const void *x, int x_dtype, int64_t tokens, int64_t x_stride, const void *weight, int weight_dtype, int64_t outer,
                            int64_t weight_stride, int64_t inner, void *x_columns, void *weight_columns, void *out, void *workspace,
                            int64_t workspace_bytes, void *stream);
int fo_mxfp4_linear_backward(const void *dy, int dy_dtype, int64_t tokens, int64_t dy_stride, int64_t outer, int64_t inner, const void *x_columns,
                             const void *weight_columns, void *dx, int dx_dtype, void *dw, int dw_dtype, void *workspace,
                             int64_t workspace_bytes, void *stream);

/*
 * What stands between the linear layers of a language model and at its two ends (no counterpart in the reference).  Rows may lie any
 * distance apart (strides in elements), their values are adjacent.
 *
 * Root-mean-square norm of the rows of s = x + residual (rounded to the residual's type and written to out_stream; s = x where
 * residual is NULL):  y = s / sqrt(mean(s^2) + eps) * weight.  x and y are of x_dtype, residual and out_stream of stream_dtype (x_dtype or
 * fp32), weight of any type or NULL (ones); y and out_stream are contiguous.  inverse (NULL, or `rows` fp32 numbers) gets
 * 1 / sqrt(mean(s^2) + eps), which the backward pass takes.  The second form writes y, in fp32 up to there, in MXFP4 as
 * fo_mxfp4_quantize lays it out.
 */
#define FO_RMS_NORM_MOST_COLS 16384
int fo_rms_norm(const void *x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void *residual, int stream_dtype,
                int64_t residual_stride, const void *weight, int weight_dtype, float eps, void *out_stream, void *y, float *inverse,
                void *stream);
int fo_rms_norm_mxfp4(const void *x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void *residual, int stream_dtype,
                      int64_t residual_stride, const void *weight, int weight_dtype, float eps, void *out_stream, void *codes, void *scales,
                      void *stream);

/* Gradients.  s: the stream (x where there was no residual, stream_dtype = x_dtype then); dy of x_dtype; dstream: the gradient that the stream itself
 * has, or NULL.  dx (x_dtype) and dresidual (stream_dtype), contiguous, get the same values, dw those of weight; any may be NULL.
 * dw needs a workspace of fo_rms_norm_backward_workspace bytes of device memory, aligned to 16. */
int64_t fo_rms_norm_backward_workspace(int64_t rows, int64_t cols);
int fo_rms_norm_backward(const void *s, int stream_dtype, int64_t s_stride, const void *weight, int weight_dtype, const float *inverse,
                         const void *dy, int x_dtype, int64_t dy_stride, const void *dstream, int64_t dstream_stride, int64_t rows,
                         int64_t cols, void *dx, void *dresidual, void *dw, void *workspace, int64_t workspace_bytes, void *stream);

/*
 * Rows of an embedding matrix:  y[i] = scale * weight[tokens[i]], rounded once.  tokens: index_bytes 4 or 8 each, contiguous; weight:
 * vocabulary x cols of `dtype`; y contiguous.  A token outside 0 .. vocabulary - 1 makes a row of NaNs.
 * The gradient of the matrix (vocabulary x cols, contiguous):  dw[v] = scale * sum of dy[i] over the i with tokens[i] = v, in fp32 and a fixed
 * order, rounded once; rows of no token are zero, and so is row `padding` (-1: none); tokens outside the vocabulary are left out.
 * workspace: fo_embedding_backward_workspace bytes of device memory, aligned to 256.
 */
#define FO_EMBEDDING_MOST_TOKENS 33554432
#define FO_EMBEDDING_MOST_ROWS 8388607 /* of the matrix */
int fo_embedding(const void *tokens, int index_bytes, int64_t n_tokens, const void *weight, int dtype, int64_t vocabulary, int64_t cols,
                 int64_t weight_stride, float scale, void *y, void *stream);
int64_t fo_embedding_backward_workspace(int64_t n_tokens, int64_t vocabulary, int64_t cols);
int fo_embedding_backward(const void *tokens, int index_bytes, int64_t n_tokens, const void *dy, int dtype, int64_t dy_stride, int64_t vocabulary,
                          int64_t cols, float scale, int64_t padding, void *dw, void *workspace, int64_t workspace_bytes, void *stream);

/*
 * Cross entropy of the logits x weight' (tokens x vocabulary, never in memory) against target tokens:
 *     loss[i] = log sum exp(logits[i]) - (1 - smoothing) logits[i][target[i]] - smoothing mean(logits[i]),     0 where target[i] = ignore
 * x: tokens x cols, weight: vocabulary x cols, both of `dtype`; targets: index_bytes 4 or 8 each, contiguous.  A target outside the
 * vocabulary makes a NaN.
 *   loss: fp32, `tokens` of them, or one: their sum or their sum over the number of targets that are not ignored
 *   kept: FO_LINEAR_CROSS_ENTROPY_KEPT fp32 numbers that the backward pass takes: of each row the largest logit, of each the log of the sum of exp(logit - largest), the
 *   number of targets that are not ignored, and the rows' targets as int32 (-1: ignored, -2: none of the vocabulary; anything else outside the vocabulary
 *   is read as no target)
 * Backward: upstream: the loss's gradient, fp32, upstream_stride elements apart (0: one for all); dx (tokens x cols) and dw (vocabulary
 * x cols) of `dtype`, contiguous, either may be NULL.  workspace: device memory, aligned to 256; its size goes by the operands' addresses and
 * strides too (what the matrix cores cannot read in place is laid out there).
 */
#define FO_LINEAR_CROSS_ENTROPY_KEPT(tokens) (3 * (tokens) + 1)
enum fo_reduction { FO_REDUCE_NONE = 0, FO_REDUCE_SUM = 1, FO_REDUCE_MEAN = 2 };
int64_t fo_linear_cross_entropy_workspace(const void *x, int dtype, int64_t tokens, int64_t x_stride, const void *weight, int64_t weight_stride,
                                          int64_t vocabulary, int64_t cols, float smoothing);
int fo_linear_cross_entropy(const void *x, int dtype, int64_t tokens, int64_t x_stride, const void *weight, int64_t weight_stride,
                            int64_t vocabulary, int64_t cols, const void *targets, int index_bytes, int64_t ignore, int reduction,
                            float smoothing, float *loss, float *kept, void *workspace, int64_t workspace_bytes, void *stream);
int64_t fo_linear_cross_entropy_backward_workspace(const void *x, int dtype, int64_t tokens, int64_t x_stride, const void *weight,
                                                   int64_t weight_stride, int64_t vocabulary, int64_t cols, int want_dx, int want_dw);
int fo_linear_cross_entropy_backward(const void *x, int dtype, int64_t tokens, int64_t x_stride, const void *weight, int64_t weight_stride,
                                     int64_t vocabulary, int64_t cols, int reduction, float smoothing, const float *kept,
                                     const float *upstream, int64_t upstream_stride, void *dx, void *dw, void *workspace,
                                     int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* FLASHOPTIM_HIP_H */
