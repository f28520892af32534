/*
 * battgp_products.h - C-ABI of libbattgp_products.so: matrix products next to the exact-GP engine's own
 * (bgp_gemm_nt_async_dev of battgp.h: one pair of operands, fp64), for MI355X (gfx950).
 *
 * Conventions
 *   - no handle and no memory of the library's own: every call names its device and the HIP stream
 *     (a hipStream_t, NULL = the device's default stream) it enqueues its kernels on, returns without waiting,
 *     and may be captured into a graph.  Calls may come from several threads at once;
 *   - pointers are device pointers on that device.  Matrices are row-major: element (i, j) of A is A[i * lda + j],
 *     leading dimensions and strides in elements.  Any alignment of the element type will do; 16-byte alignment of the
 *     base and of each row is faster;
 *   - an output overlaps no input, except where noted;
 *   - return value: 0 ok, -1 bad argument (nothing was enqueued), -2 HIP error; text in bgp_products_last_error();
 *   - a product that takes a workspace returns the bytes it needs (> 0, nothing was enqueued) where it is given fewer or
 *     NULL; call it again with that much.  The need depends on types, sizes, strides and alignment only.  The workspace
 *     (16-byte aligned) is free again behind the call's kernels on its stream: calls on one stream may share one,
 *     concurrent ones may not.  It holds copies of operands in aligned rows and partial sums, never anything that the
 *     next call would use.
 */
#ifndef BATTGP_PRODUCTS_H
#define BATTGP_PRODUCTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { BGP_F64 = 0, BGP_F32 = 1, BGP_BF16 = 2, BGP_F16 = 3 };

#define BGP_MAX_GROUPS 65535
#define BGP_INT8_MAX_K 131071 /* 128 * 128 * K < 2^31 */

/* Text of the calling thread's last error ("" if none). */
const char* bgp_products_last_error(void);

/* Products grouped by expert, ragged sizes.  Row t of X[T, K] belongs to group g where offsets[g] <= t < offsets[g + 1]:
 *   Y[t, n] = sum_k X[t, k] W_g[n, k]           n < N
 * W_g[n, k] = W[g * strideW + n * ldw + k], or W[g * strideW + k * ldw + n] with w_trans != 0; strideW = 0 gives all
 * groups the same weights.  offsets[G + 1] lies on the device, ascending, in [0, T] (values outside are clamped);
 * groups may be empty.  Rows in no group are set to 0 with zero_rest != 0 and left as they are otherwise; with G = 0 that is
 * every row, and X and W are not read (NULL will do).
 * All of one type; sums in fp32 (fp64 for BGP_F64), rounded once.
 * The gradient with respect to X is the same product of dY[T, N] with w_trans turned round (and N, K exchanged). */
int64_t bgp_grouped_gemm(int device, void* stream, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* X, int64_t ldx, const void* W,
                     int64_t strideW, int64_t ldw, int w_trans, const int64_t* offsets, void* Y, int64_t ldy, int zero_rest, void* workspace, int64_t workspace_bytes);

/* The gradient with respect to the weights:  dW_g[n, k] = sum over the rows t of g of dY[t, n] X[t, k], 0 for an empty
 * group; element (n, k) at dW[g * strideW + n * ldw + k]. */
int64_t bgp_grouped_gemm_dw(int device, void* stream, int dtype, int64_t T, int64_t N, int64_t K, int64_t G, const void* dY, int64_t lddy, const void* X,
                        int64_t ldx, const int64_t* offsets, void* dW, int64_t strideW, int64_t ldw, void* workspace, int64_t workspace_bytes);

/* x[M, K] -> codes q[M, K] in [-127, 127] and a scale for each row (fp64 for BGP_F64, else fp32):
 *   scale = max_k |x[i, k]| / 127 rounded to its type, or with pow2 != 0 the smallest power of two p with max <= 127 p;
 *           at least the smallest normal number of its type
 *   q     = x / scale rounded to the nearest whole number, ties to even
 *   rest  = x - scale * q, if not NULL (exact where the scale is a power of two): what the next slice starts from;
 *           rest == x (ldr == ldx) is allowed
 * A row that holds an infinity or a NaN gets that as its scale, codes 0 and NaN for its rest. */
int bgp_quantize_rows(int device, void* stream, int dtype, int64_t M, int64_t K, const void* x, int64_t ldx, int8_t* q, int64_t ldq, void* scale, int pow2,
                      void* rest, int64_t ldr);

/* Y[i, j] = (C[i, j] +) scale_a[i] scale_b[j] sum_k A[i, k] B[j, k]  for A[M, K], B[N, K] in 8-bit integers.
 * dtype: the type of Y and C; the scales are fp64 for BGP_F64, else fp32.  The sum is exact in 32 bits (hence
 * K <= BGP_INT8_MAX_K), what follows is computed in fp64 and rounded once.  C may be NULL; C == Y (ldc == ldy) is allowed. */
int64_t bgp_int8_gemm(int device, void* stream, int dtype, int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb,
                  const void* scale_a, const void* scale_b, const void* C, int64_t ldc, void* Y, int64_t ldy, void* workspace,
                  int64_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* BATTGP_PRODUCTS_H */
