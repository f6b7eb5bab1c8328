// Arguments and launchers shared by the grouped-product translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kmcts_grouped.h"
#include "kmcts_internal.h"

namespace kmcts {
namespace grouped {

// Y = X W_e^T or X W_e by group (dense: ends == nullptr, groups 1).
struct ForwardArgs {
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t w_stride, ldw;
    void* y;
    int64_t ldy;
    const int32_t* ends;
    int groups, rows, n, k;
    bool zero_rest;
    // MXFP4 operands only.
    const uint8_t* x_scales;
    int64_t ldxs;
    const uint8_t* w_scales;
    int64_t ws_stride, ldws;
};

struct WgradArgs {
    const void* dy;
    int64_t lddy;
    const void* x;
    int64_t ldx;
    void* dw;
    int64_t dw_stride, lddw;
    bool fp32, accumulate;
    const int32_t* ends;
    int groups, rows, n, k;
};

// Fills in a launch attribute: the grid's blocks may start before the grids
// ahead of it in the stream have finished; its kernel waits for them itself.
inline void allow_early_start(cudaLaunchAttribute* attr) {
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
}

enum class Operand { kBf16Col, kBf16Row, kMxfp4 };

// The tensor-core launchers return KMCTS_ENOTSUP, having launched nothing, for
// operands that TMA cannot address.
int launch_forward_pair(const ForwardArgs& a, Operand kind, uint64_t limit_ns, cudaStream_t stream, int* status);
int launch_forward_split(const ForwardArgs& a, Operand kind, int splits, uint64_t limit_ns, cudaStream_t stream,
                         int* status);
int launch_wgrad_pair(const WgradArgs& a, uint64_t limit_ns, cudaStream_t stream, int* status);

int launch_forward_simt(const ForwardArgs& a, Operand kind, cudaStream_t stream);
int launch_wgrad_simt(const WgradArgs& a, cudaStream_t stream);

}  // namespace grouped
}  // namespace kmcts
