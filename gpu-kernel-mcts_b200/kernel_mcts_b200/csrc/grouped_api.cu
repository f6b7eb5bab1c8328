// C entry points of the grouped products (declared in include/kmcts_grouped.h).
#include "grouped_internal.h"

using namespace kmcts;
using namespace kmcts::grouped;

namespace {

bool bad_groups(const int32_t* ends, int groups, int rows, int n, int k) {
    return rows < 0 || n < 0 || k < 0 || groups < 1 || groups > KMCTS_MAX_GROUPS || !ends;
}

int forward(const ForwardArgs& a, Operand kind, int kernel, cudaStream_t stream, int* status) {
    if (a.rows == 0 || a.n == 0) return KMCTS_OK;
    (void)status;
    if (kernel != KMCTS_KERNEL_AUTO && kernel != KMCTS_KERNEL_SIMT) return KMCTS_ENOTSUP;
    return launch_forward_simt(a, kind, stream);
}

}  // namespace

extern "C" {

int kmcts_bf16_grouped_gemm(const void* X, int64_t ldx, const void* W, int64_t w_stride, int64_t ldw, int w_layout,
                            void* Y, int64_t ldy, const int32_t* ends, int groups, int rows, int N, int K, int flags,
                            int kernel, void* stream, int* device_status) {
    if (bad_groups(ends, groups, rows, N, K)) return KMCTS_EINVAL;
    if (w_layout != KMCTS_B_COL && w_layout != KMCTS_B_ROW) return KMCTS_EINVAL;
    if (rows > 0 && N > 0 && (!Y || ldy < N || (K > 0 && (!X || !W || ldx < K)))) return KMCTS_EINVAL;
    if (ldw < (w_layout == KMCTS_B_COL ? K : N) || w_stride < 0) return KMCTS_EINVAL;
    ForwardArgs a = {};
    a.x = X, a.ldx = ldx;
    a.w = W, a.w_stride = w_stride, a.ldw = ldw;
    a.y = Y, a.ldy = ldy;
    a.ends = ends, a.groups = groups, a.rows = rows, a.n = N, a.k = K;
    a.zero_rest = (flags & KMCTS_GROUPED_ZERO_REST) != 0;
    return forward(a, w_layout == KMCTS_B_COL ? Operand::kBf16Col : Operand::kBf16Row, kernel,
                   static_cast<cudaStream_t>(stream), device_status);
}

int kmcts_bf16_grouped_wgrad(const void* dY, int64_t lddy, const void* X, int64_t ldx, void* dW, int64_t dw_stride,
                             int64_t lddw, int dw_type, int accumulate, const int32_t* ends, int groups, int rows,
                             int N, int K, int kernel, void* stream, int* device_status) {
    if (bad_groups(ends, groups, rows, N, K)) return KMCTS_EINVAL;
    if (dw_type != KMCTS_TYPE_BF16 && dw_type != KMCTS_TYPE_FP32) return KMCTS_EINVAL;
    if (accumulate && dw_type != KMCTS_TYPE_FP32) return KMCTS_EINVAL;
    if (N == 0 || K == 0) return KMCTS_OK;
    if (!dW || lddw < K || dw_stride < 0 || (rows > 0 && (!dY || !X || lddy < N || ldx < K))) return KMCTS_EINVAL;
    WgradArgs a = {};
    a.dy = dY, a.lddy = lddy;
    a.x = X, a.ldx = ldx;
    a.dw = dW, a.dw_stride = dw_stride, a.lddw = lddw;
    a.fp32 = dw_type == KMCTS_TYPE_FP32, a.accumulate = accumulate != 0;
    a.ends = ends, a.groups = groups, a.rows = rows, a.n = N, a.k = K;
    (void)device_status;
    if (kernel != KMCTS_KERNEL_AUTO && kernel != KMCTS_KERNEL_SIMT) return KMCTS_ENOTSUP;
    return launch_wgrad_simt(a, static_cast<cudaStream_t>(stream));
}

int kmcts_mxfp4_gemm(const void* A, int64_t lda, const void* A_scales, int64_t ldas, const void* B, int64_t b_stride,
                     int64_t ldb, const void* B_scales, int64_t bs_stride, int64_t ldbs, void* Y, int64_t ldy,
                     const int32_t* ends, int groups, int rows, int N, int K, int flags, int kernel, void* stream,
                     int* device_status) {
    if (rows < 0 || N < 0 || K < 0 || K % 32 != 0 || groups < 1 || groups > KMCTS_MAX_GROUPS) return KMCTS_EINVAL;
    if (!ends && groups != 1) return KMCTS_EINVAL;
    if (rows > 0 && N > 0 && (!Y || ldy < N)) return KMCTS_EINVAL;
    if (rows > 0 && N > 0 && K > 0 && (!A || !A_scales || !B || !B_scales)) return KMCTS_EINVAL;
    if (lda < K / 2 || ldb < K / 2 || ldas < K / 32 || ldbs < K / 32 || b_stride < 0 || bs_stride < 0)
        return KMCTS_EINVAL;
    ForwardArgs a = {};
    a.x = A, a.ldx = lda;
    a.w = B, a.w_stride = b_stride, a.ldw = ldb;
    a.y = Y, a.ldy = ldy;
    a.ends = ends, a.groups = groups, a.rows = rows, a.n = N, a.k = K;
    a.zero_rest = (flags & KMCTS_GROUPED_ZERO_REST) != 0;
    a.x_scales = static_cast<const uint8_t*>(A_scales), a.ldxs = ldas;
    a.w_scales = static_cast<const uint8_t*>(B_scales), a.ws_stride = bs_stride, a.ldws = ldbs;
    return forward(a, Operand::kMxfp4, kernel, static_cast<cudaStream_t>(stream), device_status);
}

}  // extern "C"
