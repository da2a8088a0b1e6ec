/*
 * uh_model_ops.h -- C ABI of the operators around the regressor on MI355X (gfx950): what its optimizer step needs beside
 * Adam (the global norm of many gradient tensors, clipping by it, the Adam update that clips on the way), and the 8-bit
 * integer products of its fully connected head for evaluation.  Library: lib/libuh_model_ops.so.
 *
 * Conventions (those of uh_hotpath.h)
 *   - tensor pointers are DEVICE pointers owned by the caller; arrays of pointers, lengths and types are HOST arrays, read
 *     during the call only.
 *   - every call only ENQUEUES work on `stream` (hipStream_t as void*; NULL = default stream) and returns; nothing allocates or
 *     frees device memory, nothing synchronises, nothing is kept between calls.  Every call can be captured into a hipGraph;
 *     a workspace must not be in use by two calls at once.
 *   - the device that owns the tensors has to be the current one.
 *   - entry points are thread-safe; they neither throw nor abort.
 *   - return value: 0 = ok; > 0 = a hipError_t of the launch; < 0 = argument error.  After an argument error nothing was enqueued.
 *   - results do not depend on timing: sums are added in a fixed order (or are sums of integers).
 */
#ifndef UH_MODEL_OPS_H
#define UH_MODEL_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define UHM_ABI_VERSION 1

#if defined(__GNUC__)
#define UHM_API __attribute__((visibility("default")))
#else
#define UHM_API
#endif

/* argument errors (the first five as in uh_hotpath.h) */
#define UHM_E_NULL        (-1)   /* a required pointer is NULL */
#define UHM_E_SHAPE       (-2)   /* a negative or inconsistent dimension, an empty list */
#define UHM_E_WORKSPACE   (-4)   /* workspace missing or smaller than *_workspace_bytes() */
#define UHM_E_TOO_LARGE   (-5)   /* a dimension outside what the kernels index, or a sum that 32 bits may not hold */
#define UHM_E_DTYPE       (-7)   /* unknown element type */
#define UHM_E_OVERLAP     (-8)   /* memory that is written overlaps other memory of the call */
#define UHM_E_ALIGN       (-9)   /* pointer or stride not aligned as required */
#define UHM_E_VALUE       (-10)  /* a scalar argument outside its range */
#define UHM_E_HOST_MEMORY (-11)  /* out of host memory */

/* element types */
#define UHM_F32  0
#define UHM_BF16 1
#define UHM_F16  2

typedef void* uhm_stream_t;      /* hipStream_t */

UHM_API int         uhm_abi_version(void);
UHM_API const char* uhm_error_string(int code);

/* ---- global norm, clipping, clipped Adam -------------------------------------------------------------------------------
 * A list is `count` >= 1 tensors of numel[i] >= 0 contiguous elements of type dtypes[i], each at least element-aligned (16-byte
 * aligned tensors go faster).  numel[i] == 0 tensors are skipped (their pointer may be NULL).  Up to 2^31 - 1 chunks of 4096
 * elements per list.  Sums of squares are held in f64, so that none over- or underflows on the way; the norm is told in f32, and one
 * above FLT_MAX (100 values of 3e38) is infinite there: it counts as not finite.
 * Workspace: uhm_multi_workspace_bytes(count) bytes, 8-byte aligned.  It overlaps neither the tensors nor a norm of the call.   */
UHM_API size_t uhm_multi_workspace_bytes(int count);

/* norm[0] = sqrt(sum_i sum_j tensors[i][j]^2), f32.  Tensors may overlap each other (each counts), norm none of them.        */
UHM_API int uhm_global_norm(const void* const* tensors, const long long* numel, const int* dtypes, int count, float* norm,
                            void* workspace, size_t workspace_bytes, uhm_stream_t stream);

/* out[i] = tensors[i] * f,  f = clip_norm / n if n > clip_norm, else 1; NaN if n is not finite (as tf.clip_by_global_norm: every
 * value becomes NaN).  n = use_norm[0] when use_norm (a device scalar) is given, else the global norm; norm[0] <- n (norm may
 * be NULL).  A factor below the normal range of f32 keeps its bits.  out[i] may equal tensors[i] (in place; with f = 1 nothing is then written); any other overlap of an output is
 * UHM_E_OVERLAP, of norm and use_norm too (they may be the same).  0 < clip_norm (may be +inf).  Workspace may be NULL when use_norm
 * is given.                                */
UHM_API int uhm_clip_by_global_norm(const void* const* tensors, void* const* out, const long long* numel, const int* dtypes,
                                    int count, float clip_norm, const float* use_norm, float* norm, void* workspace,
                                    size_t workspace_bytes, uhm_stream_t stream);

/* One Adam step on f32 variables from gradients of type grad_dtypes[i], clipped on the way (the gradients are not written):
 *   n, f as above (n = use_norm[0] when it is given);  g = f * grad;  m <- beta1 m + (1 - beta1) g;  v <- beta2 v + (1 - beta2) g^2;
 *   p <- p - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * step >= 1 is the number of this update.  With UHM_SKIP_NONFINITE a norm that is not finite leaves p, m and v as they are
 * (otherwise they become NaN).  norm[0] <- n (may be NULL).  No overlap among params, m, v and with the gradients.          */
#define UHM_SKIP_NONFINITE 1u
UHM_API int uhm_adam_clip_update(float* const* params, const void* const* grads, float* const* exp_avgs,
                                 float* const* exp_avg_sqs, const long long* numel, const int* grad_dtypes, int count,
                                 double lr, double beta1, double beta2, double eps, long long step, float clip_norm,
                                 unsigned flags, const float* use_norm, float* norm, void* workspace, size_t workspace_bytes, uhm_stream_t stream);

/* ---- products in 8-bit integers ---------------------------------------------------------------------------------------------
 * A matrix of rows in 8 bits: int8 [rows, K] with row stride ld (bytes; ld % 16 == 0, K <= ld <= 2^23), 16-byte aligned, and one f32
 * scale per row; the value at (r, k) is q[r * ld + k] * scale[r].  Every row must be READABLE up to K rounded up to a multiple
 * of 16; what stands behind K does not matter.  Sums are exact in 32-bit integers: 1 <= K <= 131071 (131071 * 128^2 < 2^31).  */

/* Rows of f32 / bf16 / f16 x [rows, K] (row stride x_ld in elements) -> q, scale, symmetric around 0:
 *   top = max |x_r|;  scale = top / 127;  q = round_to_nearest_even(x * (127 / top)), the quotients rounded to f32, the product
 *   exact.  A row whose top is below 2^-120 gets q = 0 and scale 0; one that holds an infinity or NaN gets q = 0 and scale NaN
 *   (every product with it is NaN).  q is written up to K rounded up to 16, zeros behind K;
 *   x, q and scale do not overlap.                                 */
UHM_API int uhm_quantize_rows(const void* x, int dtype, long long x_ld, int8_t* q, long long q_ld, float* scale, long long rows,
                              long long K, uhm_stream_t stream);

/* out [M, N] (contiguous, out_dtype) = act((a . b^T) * a_scale_m * b_scale_n + bias_n): a [M, K] the tokens, b [N, K] the
 * channels of a weight; bias [N] f32 or NULL; act = max(., 0) with UHM_RELU (NaN stays NaN).  M, N >= 0;
 * out overlaps none of the operands, and what is needed of the workspace neither them nor out; at most 2^22 blocks of 32 x 64
 * outputs and 2^27 channels.
 * Few rows: the sum over K is split over blocks and joined in integers through `workspace` (uhm_int8_matmul_workspace_bytes,
 * may be 0 and NULL then; 16-byte aligned).                                                                                  */
#define UHM_RELU 1u
UHM_API size_t uhm_int8_matmul_workspace_bytes(long long M, long long N, long long K);
UHM_API int uhm_int8_matmul(const int8_t* a, long long a_ld, const float* a_scale, const int8_t* b, long long b_ld,
                            const float* b_scale, const float* bias, void* out, int out_dtype, long long M, long long N, long long K,
                            unsigned flags, void* workspace, size_t workspace_bytes, uhm_stream_t stream);

/* The layer on float tokens: rows of x [M, K] (row stride x_ld in elements) quantised as uhm_quantize_rows does, the product as
 * uhm_int8_matmul computes it (the same bits), out [M, N] of x's type.  One row: a single launch.  Workspace: 16-byte aligned.   */
UHM_API size_t uhm_int8_linear_workspace_bytes(long long M, long long N, long long K);
UHM_API int uhm_int8_linear(const void* x, int dtype, long long x_ld, const int8_t* b, long long b_ld, const float* b_scale,
                            const float* bias, void* out, long long M, long long N, long long K, unsigned flags, void* workspace,
                            size_t workspace_bytes, uhm_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* UH_MODEL_OPS_H */
