// C entry points of the grouped products (declared in include/kmcts_grouped.h).
#include <cudaTypedefs.h>

#include <mutex>

#include "grouped_tiles.cuh"

namespace kmcts {
namespace grouped {

bool encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims,
                const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle) {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    std::call_once(once, [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult query;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &query) ==
                cudaSuccess &&
            query == cudaDriverEntryPointSuccess)
            encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(entry);
    });
    const cuuint32_t steps[3] = {1, 1, 1};
    cuuint64_t d[3], s[2];
    cuuint32_t b[3];
    for (int i = 0; i < rank; ++i) d[i] = dims[i], b[i] = box[i];
    for (int i = 0; i + 1 < rank; ++i) s[i] = strides[i];
    return encode && encode(map, type, rank, const_cast<void*>(base), d, s, b, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
                         CUDA_SUCCESS;
}

bool encode_forward_maps(const ForwardArgs& f, Operand operand, CUtensorMap* w, CUtensorMap (&x)[3],
                         const uint32_t (&box_rows)[3]) {
    const bool mx = operand == Operand::kMxfp4, row = operand == Operand::kBf16Row;
    const auto type = mx ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t size = mx ? 1 : 2, n = f.n;
    const uint64_t k = mx ? f.k / 2 : f.k;  // contiguous elements of a row
    const uint32_t inner = mx ? 128 : 64;   // 128 bytes
    {
        const uint64_t group = f.groups > 1 ? f.w_stride : f.ldw * (row ? k : n);
        const uint64_t dims[3] = {row ? n : k, row ? k : n, static_cast<uint64_t>(f.groups)};
        const uint64_t strides[2] = {f.ldw * size, group * size};
        const uint32_t box[3] = {inner, row ? 64u : 128u, 1};
        if (!encode_map(w, type, 3, f.w, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return false;
    }
    const uint64_t dims[2] = {k, static_cast<uint64_t>(f.rows)}, strides[1] = {f.ldx * size};
    for (int i = 0; i < 3; ++i) {
        const uint32_t box[2] = {inner, box_rows[i]};
        if (!encode_map(&x[i], type, 2, f.x, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return false;
    }
    return true;
}

void scale_spans(const ForwardArgs& f, ScaleSpan* x, ScaleSpan* w) {
    *x = *w = {nullptr, nullptr};
    if (f.x_scales == nullptr) return;
    *x = {f.x_scales, f.x_scales + (f.rows - 1) * f.ldxs + f.k / 32};
    *w = {f.w_scales, f.w_scales + (f.groups - 1) * f.ws_stride + (f.n - 1) * f.ldws + f.k / 32};
}

}  // namespace grouped
}  // namespace kmcts

using namespace kmcts;
using namespace kmcts::grouped;

namespace {

// Sizes leave room to round up to whole tiles.
constexpr int kMaxSize = 0x7fffffff - 1023;

bool bad_sizes(int groups, int rows, int n, int k) {
    return rows < 0 || n < 0 || k < 0 || rows > kMaxSize || n > kMaxSize || k > kMaxSize || groups < 1 ||
           groups > KMCTS_MAX_GROUPS;
}

// How long a wait of a launch may last: the library's limit, and ten
// microseconds for each stage that one CTA walks through.  Epilogues and the
// gradient's tail warps sleep through the whole contraction of a tile (the tail
// warps through tiles without a tail, too), which takes 0.3 to 1.2 us a stage:
// with the limit alone, contractions of more than about 2 s were given up.  Ten
// minutes are more than any product takes whose operands fit in memory.
uint64_t wait_limit(int64_t stages) {
    constexpr uint64_t most = 600000000000ull;
    const uint64_t limit = gemm::kDefaultWaitNs + 10000ull * static_cast<uint64_t>(stages);
    return limit < most ? limit : most;
}

// Whether the few-rows kernel should take a product, and how many CTAs share
// one of its tiles (128 weight rows x 64 tokens; how many there are is known
// up to where the groups end).  GPU time on B200 with operands read from HBM,
// pair / split in two / split in four:
// * as many tiles as a quarter of the SMs or fewer: four (64 x 4096 x 4096 BF16
//   25.6 / 18.1 / 13.7 us, MXFP4 12.7 / 11.7 / 10.2);
// * up to half the SMs: two, one round of tiles (128 x 4096 x 4096 BF16 26.9 /
//   18.5 / 18.2, MXFP4 13.9 / 12.1 / 13.2; past it pairs win: 512 x 4096 x 4096
//   29.5 / 48.9 / 49.7);
// * more tiles, few rows a group on average: two, whose finer tiles share the
//   SMs evenly while the weights stream in (64 experts of 2048 x 4096, 256 rows
//   180 / 166 / 185; 16 of 4096 x 4096, 512 rows 110 / 91 / -, 768 rows 111 /
//   110, 1024 rows 111 / 117; MXFP4 32 of 2048 x 4096, 1024 rows 37.7 / 35.4,
//   1500 rows 39.0 / 42.5).
struct FewRows {
    bool better;
    int splits;
};

FewRows few_rows(const ForwardArgs& a) {
    const int64_t used = a.groups < a.rows ? a.groups : a.rows;
    const int64_t tiles = ((a.rows + 63) / 64 + used - 1) * ((a.n + 127) / 128);
    const int sms = multiprocessor_count();
    if (4 * tiles <= sms) return {true, 4};
    return {2 * tiles <= sms || a.rows <= 40LL * a.groups, 2};
}

int forward(const ForwardArgs& a, Operand kind, int kernel, cudaStream_t stream, int* status) {
    if (a.rows == 0 || a.n == 0) return KMCTS_OK;
    if (kernel < KMCTS_KERNEL_AUTO || kernel > KMCTS_KERNEL_GROUPED_SPLIT) return KMCTS_EINVAL;
    // K = 0 (all zeros) has nothing to copy in; it is left to the CUDA cores.
    if (kernel != KMCTS_KERNEL_SIMT && a.k > 0) {
        if (!status) status = default_status_ptr();
        if (!status) return KMCTS_EHANDLE;
        const FewRows few = few_rows(a);
        const bool split = kernel == KMCTS_KERNEL_GROUPED_SPLIT || (few.better && kernel != KMCTS_KERNEL_GROUPED_PAIR);
        const uint64_t limit = wait_limit(a.k / (kind == Operand::kMxfp4 ? 256 : 64) + 1);
        const int rc = split ? launch_forward_split(a, kind, few.splits, limit, stream, status)
                             : launch_forward_pair(a, kind, limit, stream, status);
        if (rc != KMCTS_ENOTSUP || kernel != KMCTS_KERNEL_AUTO) return rc;
    }
    return launch_forward_simt(a, kind, stream);
}

}  // namespace

extern "C" {

int kmcts_bf16_grouped_gemm(const void* X, int64_t ldx, const void* W, int64_t w_stride, int64_t ldw, int w_layout,
                            void* Y, int64_t ldy, const int32_t* ends, int groups, int rows, int N, int K, int flags,
                            int kernel, void* stream, int* device_status) {
    if (bad_sizes(groups, rows, N, K) || !ends) return KMCTS_EINVAL;
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
    if (bad_sizes(groups, rows, N, K) || !ends) return KMCTS_EINVAL;
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
    if (kernel < KMCTS_KERNEL_AUTO || kernel > KMCTS_KERNEL_SIMT) return KMCTS_EINVAL;
    auto s = static_cast<cudaStream_t>(stream);
    if (kernel != KMCTS_KERNEL_SIMT && rows > 0) {
        int* status = device_status ? device_status : default_status_ptr();
        if (!status) return KMCTS_EHANDLE;
        // A pair takes every 74th tile of each group in turn.
        const int64_t tiles = ((N + 255LL) / 256) * ((K + 255LL) / 256), pairs = multiprocessor_count() / 2;
        const int64_t stages = (rows / 128 + static_cast<int64_t>(groups)) * ((tiles + pairs - 1) / pairs);
        const int rc = launch_wgrad_pair(a, wait_limit(stages), s, status);
        if (rc != KMCTS_ENOTSUP || kernel != KMCTS_KERNEL_AUTO) return rc;
    }
    return launch_wgrad_simt(a, s);
}

int kmcts_mxfp4_gemm(const void* A, int64_t lda, const void* A_scales, int64_t ldas, const void* B, int64_t b_stride,
                     int64_t ldb, const void* B_scales, int64_t bs_stride, int64_t ldbs, void* Y, int64_t ldy,
                     const int32_t* ends, int groups, int rows, int N, int K, int flags, int kernel, void* stream,
                     int* device_status) {
    if (bad_sizes(groups, rows, N, K) || K % 32 != 0 || (!ends && groups != 1)) return KMCTS_EINVAL;
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
