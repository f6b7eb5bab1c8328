/*
 * kmcts_grouped.h — C ABI of the expert-layer products of
 * libkmcts_gemm_sm100.so: BF16 products grouped by expert with the weights'
 * gradient, and microscaled 4-bit (MXFP4) quantisation and products.  No
 * counterpart in the reference, which has one dense GEMM.
 *
 * Groups.  `ends` is a device array of `groups` int32 values: group e owns the
 * rows ends[e-1] (0 for e = 0) up to, not including, ends[e].  The kernels read
 * it on the device, so no call waits for it.  Ends are taken in order, each
 * clamped to [end of the group before, rows]: no value can make a kernel read
 * or write out of range.  Rows behind the last end belong to no group; they
 * are left as they were, or zeroed with KMCTS_GROUPED_ZERO_REST.  A group may
 * be empty.  At most KMCTS_MAX_GROUPS groups.
 *
 * All pointers are device pointers; strides ("ld", "stride") count elements of
 * the array they belong to (bytes for packed 4-bit codes and for scales).  The
 * innermost dimension is contiguous.  Calls are asynchronous on `stream` and
 * run on the current device; they keep nothing between calls and use no
 * workspace, so calls on different streams, and graphs that captured them,
 * may overlap.  device_status is as for kmcts_bf16_gemm_ex: a wait that gives
 * up (after two seconds, and ten microseconds more for each stage of K or of a
 * group's rows that one CTA walks through) sets it and leaves results unwritten.
 *
 * Returns KMCTS_OK, KMCTS_EINVAL (pointers, sizes, strides, groups),
 * KMCTS_ENOTSUP (the requested kernel cannot run these arguments) or
 * KMCTS_EGEMM (launch failure).
 */
#ifndef KMCTS_GROUPED_H
#define KMCTS_GROUPED_H

#include "kmcts_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KMCTS_MAX_GROUPS 1024

#define KMCTS_GROUPED_ZERO_REST 1 /* flags: zero the rows behind the last group */

/* kernel: KMCTS_KERNEL_AUTO picks by size and alignment, KMCTS_KERNEL_TCGEN05
 * by size among the tensor-core kernels, KMCTS_KERNEL_SIMT is the CUDA-core
 * kernel, which takes any stride and alignment.  The forward products have two
 * tensor-core kernels: CTA pairs, and clusters that split K for few rows. */
#define KMCTS_KERNEL_GROUPED_PAIR 3
#define KMCTS_KERNEL_GROUPED_SPLIT 4

/* Element types of quantiser inputs, restored values and gradients. */
#define KMCTS_TYPE_BF16 0
#define KMCTS_TYPE_FP16 1
#define KMCTS_TYPE_FP32 2

/* Y[t, :] = X[t, :] * W_e^T (KMCTS_B_COL: W_e is [N, K] row-major) or
 * X[t, :] * W_e (KMCTS_B_ROW: W_e is [K, N] row-major) for the rows t of
 * group e; X is [rows, K], Y [rows, N], all BF16, FP32 sums rounded once.
 * With KMCTS_B_ROW on the weight of a KMCTS_B_COL product this is that
 * product's input gradient.  W_e starts at W + e * w_stride, its rows are ldw
 * apart.  The tensor-core kernels need 16-byte aligned X and W, and ldx, ldw
 * and w_stride multiples of 8. */
int kmcts_bf16_grouped_gemm(const void* X, int64_t ldx, const void* W, int64_t w_stride, int64_t ldw, int w_layout,
                            void* Y, int64_t ldy, const int32_t* ends, int groups, int rows, int N, int K, int flags,
                            int kernel, void* stream, int* device_status);

/* dW_e = dY_e^T * X_e over the rows of group e: dY is [rows, N], X [rows, K]
 * (BF16), dW_e [N, K] at dW + e * dw_stride in dw_type (KMCTS_TYPE_BF16 or
 * KMCTS_TYPE_FP32), FP32 sums.  accumulate (FP32 only) adds each sum to dW with
 * one rounding, subnormals kept, and leaves an empty group's part as it was;
 * otherwise the gradient of an empty group is zeros.  The tensor-core kernel
 * needs 16-byte aligned pointers and strides that are multiples of 16 bytes. */
int kmcts_bf16_grouped_wgrad(const void* dY, int64_t lddy, const void* X, int64_t ldx, void* dW, int64_t dw_stride,
                             int64_t lddw, int dw_type, int accumulate, const int32_t* ends, int groups, int rows,
                             int N, int K, int kernel, void* stream, int* device_status);

/* MXFP4: blocks of 32 elements along K share one E8M0 scale (a byte s that
 * stands for 2^(s - 127); 255 is NaN); elements are E2M1 codes, two a byte,
 * the even element in the low half.  K is a multiple of 32.
 *
 * Quantisation of X [rows, K] (x_type): the block's scale is 2^(floor(log2 m)
 * - 2) for its largest magnitude m, at least 2^-127; each code is the nearest
 * E2M1 value of x / scale, ties to the even code, saturating at 6.  A block
 * holding an infinity or a NaN gets the NaN scale. */
int kmcts_mxfp4_quantize(const void* X, int x_type, int64_t ldx, void* codes, int64_t ldc, void* scales, int64_t lds,
                         int64_t rows, int K, void* stream);

/* out[r, k] = value of the code times its block's scale, rounded once to
 * out_type (exact in FP32 and, from 2^-133 up, in BF16; an infinity where the
 * type ends: 2^128, in FP16 2^16). */
int kmcts_mxfp4_dequantize(const void* codes, int64_t ldc, const void* scales, int64_t lds, void* out, int out_type,
                           int64_t ldo, int64_t rows, int K, void* stream);

/* Y[t, :] = A[t, :] * B_e^T with both operands MXFP4 (A [rows, K], B_e
 * [N, K]), FP32 sums, BF16 Y.  ends == NULL: one dense product (groups 1).
 * b_stride / bs_stride: bytes from one group's codes / scales to the next. */
int kmcts_mxfp4_gemm(const void* A, int64_t lda, const void* A_scales, int64_t ldas, const void* B, int64_t b_stride,
                     int64_t ldb, const void* B_scales, int64_t bs_stride, int64_t ldbs, void* Y, int64_t ldy,
                     const int32_t* ends, int groups, int rows, int N, int K, int flags, int kernel, void* stream,
                     int* device_status);

#ifdef __cplusplus
}
#endif

#endif /* KMCTS_GROUPED_H */
