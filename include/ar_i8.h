/*
 * ar_i8.h -- C-ABI of the 8-bit path: rows held in 8 bits with a scale each, the calls that make them, read them and
 * multiply them.
 *
 * No counterpart in the reference, whose contexts compute in FP32 or FP64.  The operators stand where those of ar_hip.h
 * stand: add_rmsnorm for ar_hip_rmsnorm with the residual add ahead of it, gemm_i8 for ar_hip_dense, ar_hip_swiglu and
 * ar_hip_gemm_* (LayerFeatures.dense, domain/graph/.../layers/LayerFeatures.java:785-830; FeedForwardFeatures.feedForward,
 * engine/ml/.../FeedForwardFeatures.java:140-157), embed_i8 for the embedding copy (AutoregressiveModel.java:430).
 *
 * Same conventions as ar_hip.h: plain C, device pointers, AR_HIP_* status codes, ar_hip_last_error().  Every call
 * enqueues on the context's stream and returns; nothing is allocated.  Row counts of 0 are allowed and do nothing.
 * Outputs do not overlap inputs but where it says so.
 */
#ifndef AR_I8_H
#define AR_I8_H

#include "ar_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows in 8 bits: value (r, i) is q[r * stride + i] * scale[r].  Weights are held so by output channel (a row of the HF
 * (out, in) layout), activations by token.  Between n and the next multiple of 16 a row holds zeros: the calls below
 * write them, and of two rows that are multiplied one at least has to hold them. */
typedef struct ar_rows_i8 {
    int8_t *q;       /* 16-byte aligned; rows * stride bytes */
    float *scale;    /* [rows] */
    int64_t stride;  /* bytes from one row to the next: a multiple of 16, n .. 2^22 */
    int32_t rows;    /* 0 .. 2^24 */
    int32_t n;       /* 1 .. 131071 */
} ar_rows_i8;

/* Rows of floats to 8 bits: scale[r] = m / 127 for the largest magnitude m of x[r], q = x * (127 / m) rounded to the
 * nearest, halves to even.  A row whose largest magnitude is below 2^-100 becomes zeros with scale 0; a row that holds
 * an infinity or NaN zeros with scale NaN, which makes NaN of all that is computed from it.  x: out->rows rows of out->n
 * values of x_dtype (AR_DTYPE_F32 or AR_DTYPE_BF16), x_stride values apart (n .. 2^22). */
int ar_hip_quantize_i8(ar_hip_ctx *ctx, const void *x, int x_dtype, int x_stride, const ar_rows_i8 *out);

/* The residual's addition and its RMS norm: h[r] += x[r] (x null: nothing is added), y[r] = h[r] / sqrt(mean(h[r]^2) +
 * eps) * w.  The norm is of the sum in fp32, also where h is bf16 and keeps it rounded; squares are summed in double.
 * h, x, y: rows of n values of AR_DTYPE_F32 or AR_DTYPE_BF16 with strides as above; w fp32; eps >= 0.  y may be x itself
 * where their types and strides agree.  With eps 0 a row of zeros is NaN, and one of numbers below 2^-127 may overflow.
 * ar_hip_add_rmsnorm_i8 puts y, unrounded, into rows of 8 bits as ar_hip_quantize_i8 does: out->rows rows of out->n. */
int ar_hip_add_rmsnorm(ar_hip_ctx *ctx, void *h, int h_dtype, int h_stride, const void *x, int x_dtype, int x_stride,
                       const float *w, float eps, int rows, int n, void *y, int y_dtype, int y_stride);
int ar_hip_add_rmsnorm_i8(ar_hip_ctx *ctx, void *h, int h_dtype, int h_stride, const void *x, int x_dtype,
                          int x_stride, const float *w, float eps, const ar_rows_i8 *out);

/* Rows of 8 bits as floats: y[i] = table row tokens[i] (tokens null: row i, for count <= table->rows), of y_dtype
 * (AR_DTYPE_F32 or AR_DTYPE_BF16), y_stride values apart (n .. 2^22).  A token outside the table gives zeros.
 * count 0 .. 2^24. */
int ar_hip_embed_i8(ar_hip_ctx *ctx, const ar_rows_i8 *table, const int32_t *tokens, int count, void *y, int y_dtype,
                    int y_stride);

/* Products of rows in 8 bits, C[m][n] of A->rows x W->rows (A->n = W->n):
 *   p(W)[m][n] = A->scale[m] * W->scale[n] * sum_k A->q[m][k] * W->q[n][k]    (the sum in whole numbers, exact)
 *   AR_GEMM_STORE:    C = p(W) (+ bias[n] where bias, fp32, is given)
 *   AR_GEMM_RESIDUAL: C += p(W)
 *   AR_GEMM_SWIGLU:   C = p(W2) * silu(p(W)): W the gate's rows, W2 the up projection's, of W's sizes and stride
 * C is of c_dtype (AR_DTYPE_F32 or AR_DTYPE_BF16), ldc values apart, N .. 2^24.  A->rows * W->rows is at most 2^40.
 * The sum goes to fp32 and each scale, the addition and the gate's steps round there; a bf16 result is rounded once more.
 * Scales may be any finite numbers: what is computed on the way leaves fp32 only where a product, a gate or a result does.
 * Results do not depend on how a product is cut: the same rows give the same bits in any batch.
 * `work`: device memory of the caller's, 16-byte aligned, of at least the bytes that ar_hip_gemm_i8_work reports (null
 * where that is 0) for these very sizes: it does not grow with them (2,560 outputs over 9,728: nothing for 16 tokens, 7.9 MB
 * for 128, nothing for 509), so a caller with many sizes asks for each.  Its contents mean nothing between calls.  Calls ordered on one stream may share it, calls that may
 * run at the same time may not. */
int ar_hip_gemm_i8_work(ar_hip_ctx *ctx, int M, int N, int K, int epilogue, size_t *bytes);
int ar_hip_gemm_i8(ar_hip_ctx *ctx, const ar_rows_i8 *A, const ar_rows_i8 *W, const ar_rows_i8 *W2, const float *bias,
                   void *C, int c_dtype, int ldc, int epilogue, void *work, size_t work_bytes);

#ifdef __cplusplus
}
#endif

#endif /* AR_I8_H */
