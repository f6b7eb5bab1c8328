// The expert-layer calls on torch tensors: argument checks, allocation of
// results, the current stream, and the C call of include/kmcts_grouped.h.
//
// Through Python and ctypes such a call took 11 to 12 us on the host, longer
// than a small kernel runs; the same steps here take half of that.  Nothing is
// computed here, and there is no other route: kernel_mcts_b200/grouped.py and
// mxfp4.py call these functions.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>

#include "kmcts_grouped.h"

namespace py = pybind11;

namespace {

using at::ScalarType;
using at::Tensor;
using Types = std::initializer_list<ScalarType>;

constexpr int64_t kMaxSize = (1LL << 31) - (1LL << 10);  // 32-bit sizes with room to round up
constexpr int kBlock = 32;                               // elements that share an MXFP4 scale

// A C entry point's error code; Python sees KmctsError.
struct Failure : std::runtime_error {
    int code;
    std::string call;
    Failure(int c, std::string name)
        : std::runtime_error(name + " failed (" + std::to_string(c) + ")"), code(c), call(std::move(name)) {}
};

void check_code(int code, const char* call) {
    if (code != KMCTS_OK) throw Failure(code, call);
}

template <typename... Parts>
std::string text(const Parts&... parts) {
    std::ostringstream out;
    (out << ... << parts);
    return out.str();
}

std::string type_name(ScalarType type) {
    switch (type) {
        case ScalarType::BFloat16: return "bfloat16";
        case ScalarType::Half: return "float16";
        case ScalarType::Float: return "float32";
        case ScalarType::Byte: return "uint8";
        default: return c10::toString(type);
    }
}

std::string shape_text(at::IntArrayRef shape) {
    std::string out = "(";
    for (size_t i = 0; i < shape.size(); ++i) out += (i ? ", " : "") + std::to_string(shape[i]);
    return out + ")";
}

// Elements from one row to the next; where there is only one row, the row's
// length rounded up to `unit`, whatever stride torch reports.
int64_t row_stride(const char* name, const Tensor& t, int64_t unit) {
    const int64_t length = t.size(-1);
    if (t.size(-2) <= 1) return (length + unit - 1) / unit * unit;
    const int64_t stride = t.stride(-2);
    if (stride < length)
        throw py::value_error(text(name, " has overlapping rows (row stride ", stride, ", row length ", length, ")"));
    return stride;
}

// A tensor of one of the types on the device, its innermost dimension
// contiguous; returns its row stride.
int64_t check_rows(const char* name, const Tensor& t, int64_t dims, Types types, int device, int64_t unit) {
    bool known = false;
    for (ScalarType type : types) known |= t.scalar_type() == type;
    if (!known) {
        std::string wanted;
        for (ScalarType type : types) wanted += (wanted.empty() ? "" : " or ") + type_name(type);
        throw py::type_error(text(name, " must be ", wanted, ", got ", type_name(t.scalar_type())));
    }
    if (!t.is_cuda()) throw py::value_error(text(name, " must be a CUDA tensor"));
    if (t.get_device() != device)
        throw py::value_error(text(name, " must be on cuda:", device, ", got cuda:", static_cast<int>(t.get_device())));
    if (t.dim() != dims)
        throw py::value_error(text(name, " must have ", dims, " dimensions, got shape ", shape_text(t.sizes())));
    if (t.size(-1) > 1 && t.stride(-1) != 1)
        throw py::value_error(text(name, " must be contiguous along its last dimension"));
    return row_stride(name, t, unit);
}

void check_shape(const char* name, const Tensor& t, at::IntArrayRef shape) {
    if (t.sizes() != shape)
        throw py::value_error(text(name, " must have shape ", shape_text(shape), ", got ", shape_text(t.sizes())));
}

int cuda_index(const Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

int check_groups(const Tensor& ends, int device) {
    if (ends.scalar_type() != ScalarType::Int || ends.dim() != 1 || !ends.is_contiguous())
        throw py::type_error("ends must be a contiguous one-dimensional int32 tensor");
    if (cuda_index(ends) != device)
        throw py::value_error(text("ends must be on cuda:", device, ", got ", ends.device().str()));
    if (ends.size(0) < 1 || ends.size(0) > KMCTS_MAX_GROUPS)
        throw py::value_error(text("there must be 1 to ", KMCTS_MAX_GROUPS, " groups, got ", ends.size(0)));
    return static_cast<int>(ends.size(0));
}

void check_sizes(std::initializer_list<int64_t> sizes) {
    for (int64_t size : sizes)
        if (size > kMaxSize) throw py::value_error(text("sizes must be at most ", kMaxSize, ", got ", size));
}

int* status_pointer(const std::optional<Tensor>& status, int device) {
    if (!status) return nullptr;
    if (status->scalar_type() != ScalarType::Int || cuda_index(*status) != device || status->numel() < 1)
        throw py::value_error(text("status must be an int32 tensor on cuda:", device, " with at least one element"));
    return status->mutable_data_ptr<int>();
}

Tensor empty(at::IntArrayRef shape, ScalarType type, int device) {
    return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)),
                                  std::nullopt);
}

void* current_stream(int device) {
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

// The calls are not recorded by autograd, so what computed the tensor's earlier
// values would get a gradient for the ones written over them.
void check_writable(const char* name, const Tensor& t) {
    if (at::GradMode::is_enabled() && t.requires_grad())
        throw py::value_error(text(name, " must not require a gradient (write it under torch.no_grad())"));
}

// The caller's tensor has been written: autograd then notices where it was
// saved for a backward pass.  (Inference tensors count no versions.)
void mark_written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int i32(int64_t v) { return static_cast<int>(v); }

// ------------------------------------------------------------------- grouped

Tensor grouped_gemm(const Tensor& x, const Tensor& w, const Tensor& ends, const std::optional<Tensor>& out, int layout,
                    int kernel, const std::optional<Tensor>& status) {
    const int device = cuda_index(x);
    const int64_t ldx = check_rows("x", x, 2, {ScalarType::BFloat16}, device, 8);
    const int64_t ldw = check_rows("w", w, 3, {ScalarType::BFloat16}, device, 8);
    const int groups = check_groups(ends, device);
    const int64_t rows = x.size(0), k = x.size(1);
    const int64_t n = w.size(layout == KMCTS_B_COL ? 1 : 2), kw = w.size(layout == KMCTS_B_COL ? 2 : 1);
    if (kw != k) throw py::value_error(text("inner dimensions differ: x has K=", k, ", w has K=", kw));
    if (w.size(0) != groups) throw py::value_error(text("w holds ", w.size(0), " groups, ends ", groups));
    check_sizes({rows, n, k});
    int* const status_ptr = status_pointer(status, device);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    Tensor y;
    int64_t ldy = n;
    if (out) {
        y = *out;
        check_writable("out", y);
        ldy = check_rows("out", y, 2, {ScalarType::BFloat16}, device, 8);
        check_shape("out", y, {rows, n});
    } else {
        y = empty({rows, n}, ScalarType::BFloat16, device);
    }
    check_code(kmcts_bf16_grouped_gemm(x.const_data_ptr(), ldx, w.const_data_ptr(), groups > 1 ? w.stride(0) : 0, ldw,
                                       layout, y.mutable_data_ptr(), ldy, ends.const_data_ptr<int>(), groups, i32(rows),
                                       i32(n), i32(k), out ? 0 : KMCTS_GROUPED_ZERO_REST, kernel, current_stream(device),
                                       status_ptr),
               "kmcts_bf16_grouped_gemm");
    if (out) mark_written(y);
    return y;
}

Tensor grouped_gemm_wgrad(const Tensor& dy, const Tensor& x, const Tensor& ends, const std::optional<Tensor>& out,
                          const std::optional<ScalarType>& dtype, bool accumulate, int kernel,
                          const std::optional<Tensor>& status) {
    const int device = cuda_index(dy);
    const int64_t lddy = check_rows("dy", dy, 2, {ScalarType::BFloat16}, device, 8);
    const int64_t ldx = check_rows("x", x, 2, {ScalarType::BFloat16}, device, 8);
    const int groups = check_groups(ends, device);
    const int64_t rows = dy.size(0), n = dy.size(1), k = x.size(1);
    if (x.size(0) != rows) throw py::value_error(text("dy has ", rows, " rows, x ", x.size(0)));
    check_sizes({rows, n, k});
    const ScalarType type = dtype ? *dtype : out ? out->scalar_type() : ScalarType::BFloat16;
    if (type != ScalarType::BFloat16 && type != ScalarType::Float)
        throw py::type_error(text("the gradient must be bfloat16 or float32, got ", type_name(type)));
    if (accumulate && (!out || type != ScalarType::Float))
        throw py::value_error("accumulate needs a float32 out");
    int* const status_ptr = status_pointer(status, device);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    Tensor dw;
    int64_t ldo = k, group_stride = n * k;
    if (out) {
        dw = *out;
        check_writable("out", dw);
        ldo = check_rows("out", dw, 3, {type}, device, 8);
        check_shape("out", dw, {groups, n, k});
        group_stride = groups > 1 ? dw.stride(0) : n * ldo;
        // Groups one behind the other, or side by side in every row.
        if (groups > 1 && n > 0 && group_stride < (n - 1) * ldo + k &&
            (group_stride < k || (n > 1 && ldo < (groups - 1) * group_stride + k)))
            throw py::value_error("out has overlapping groups");
    } else {
        dw = empty({groups, n, k}, type, device);
    }
    check_code(kmcts_bf16_grouped_wgrad(dy.const_data_ptr(), lddy, x.const_data_ptr(), ldx, dw.mutable_data_ptr(),
                                        group_stride, ldo, type == ScalarType::Float ? KMCTS_TYPE_FP32 : KMCTS_TYPE_BF16,
                                        accumulate, ends.const_data_ptr<int>(), groups, i32(rows), i32(n), i32(k),
                                        kernel, current_stream(device), status_ptr),
               "kmcts_bf16_grouped_wgrad");
    if (out) mark_written(dw);
    return dw;
}

// `t` itself where the kernels can read it, else a contiguous copy (an
// expanded gradient, as a sum's backward gives, has overlapping rows).
Tensor strided_rows(const Tensor& t) {
    const bool readable = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return readable ? t : t.contiguous();
}

class GroupedLinear : public torch::autograd::Function<GroupedLinear> {
public:
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& ends,
                          int64_t layout) {
        // The gradient of each needs the other: with a frozen weight the
        // activations may go, and the other way round.
        ctx->save_for_backward({w.requires_grad() ? x : Tensor(), x.requires_grad() ? w : Tensor(), ends});
        ctx->saved_data["layout"] = layout;
        return grouped_gemm(x, w, ends, std::nullopt, i32(layout), KMCTS_KERNEL_AUTO, std::nullopt);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        // With create_graph the gradients below would not be part of it.
        if (at::GradMode::is_enabled()) throw std::runtime_error("grouped_linear is differentiable once");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &ends = saved[2];
        const int layout = i32(ctx->saved_data["layout"].toInt());
        const Tensor dy = strided_rows(grads[0]);
        Tensor dx, dw;
        if (ctx->needs_input_grad(0))
            dx = grouped_gemm(dy, w, ends, std::nullopt, layout == KMCTS_B_COL ? KMCTS_B_ROW : KMCTS_B_COL,
                              KMCTS_KERNEL_AUTO, std::nullopt);
        if (ctx->needs_input_grad(1)) {
            const bool col = layout == KMCTS_B_COL;
            dw = grouped_gemm_wgrad(col ? dy : x, col ? x : dy, ends, std::nullopt, std::nullopt, false,
                                    KMCTS_KERNEL_AUTO, std::nullopt);
        }
        return {dx, dw, Tensor(), Tensor()};
    }
};

Tensor grouped_linear(const Tensor& x, const Tensor& w, const Tensor& ends, int layout) {
    return GroupedLinear::apply(x, w, ends, static_cast<int64_t>(layout));
}

// -------------------------------------------------------------------- MXFP4

int element_code(ScalarType type) {
    return type == ScalarType::BFloat16 ? KMCTS_TYPE_BF16 : type == ScalarType::Half ? KMCTS_TYPE_FP16 : KMCTS_TYPE_FP32;
}

constexpr ScalarType kCodes[2] = {ScalarType::Byte, ScalarType::Float4_e2m1fn_x2};

// The tensor as rows of its last dimension.
Tensor as_rows(const char* name, const Tensor& t) {
    if (t.dim() == 2) return t;
    if (t.dim() < 1 || !t.is_contiguous()) throw py::value_error(text(name, " must be two-dimensional or contiguous"));
    const int64_t length = t.size(-1);
    return t.view({length ? t.numel() / length : 0, length});
}

struct PairStrides {
    int64_t codes, scales;  // row strides
};

PairStrides check_pair(const char* name, const Tensor& codes, const Tensor& scales, int64_t dims, int device) {
    const std::string codes_name = text(name, " codes"), scales_name = text(name, " scales");
    const PairStrides out = {check_rows(codes_name.c_str(), codes, dims, {kCodes[0], kCodes[1]}, device, 16),
                             check_rows(scales_name.c_str(), scales, dims, {ScalarType::Byte, ScalarType::Float8_e8m0fnu},
                                        device, 1)};
    if (codes.size(-1) % (kBlock / 2) != 0)
        throw py::value_error(text(name, " has K=", 2 * codes.size(-1), ", not a multiple of ", kBlock));
    bool same = scales.size(-1) == codes.size(-1) / (kBlock / 2);
    for (int64_t d = 0; d + 1 < dims; ++d) same &= scales.size(d) == codes.size(d);
    if (!same) {
        std::vector<int64_t> wanted = codes.sizes().vec();
        wanted.back() /= kBlock / 2;
        throw py::value_error(
            text(scales_name, " must have shape ", shape_text(wanted), ", got ", shape_text(scales.sizes())));
    }
    return out;
}

std::tuple<Tensor, Tensor> mxfp4_quantize(const Tensor& x, const std::optional<Tensor>& out_codes,
                                          const std::optional<Tensor>& out_scales) {
    if (out_codes.has_value() != out_scales.has_value()) throw py::value_error("out must hold both codes and scales");
    if (x.dim() < 1 || x.size(-1) % kBlock != 0)
        throw py::value_error(text("x must have a last dimension that is a multiple of ", kBlock, ", got shape ",
                                   shape_text(x.sizes())));
    const int device = cuda_index(x);
    const Tensor flat = as_rows("x", x);
    const int64_t ldx = check_rows("x", flat, 2, {ScalarType::BFloat16, ScalarType::Half, ScalarType::Float}, device, kBlock);
    const int64_t rows = flat.size(0), k = flat.size(1);
    check_sizes({k});
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    Tensor codes, scales, code_rows, scale_rows;
    PairStrides strides = {k / 2, k / kBlock};
    if (out_codes) {
        codes = *out_codes, scales = *out_scales;
        code_rows = as_rows("out codes", codes), scale_rows = as_rows("out scales", scales);
        strides = check_pair("out", code_rows, scale_rows, 2, device);
        std::vector<int64_t> shape = codes.sizes().vec();
        shape.back() *= 2;
        if (x.sizes() != at::IntArrayRef(shape))
            throw py::value_error(text("out must have shape ", shape_text(x.sizes()), ", got ", shape_text(shape)));
    } else {
        c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = k / 2;
        code_rows = codes = empty(shape, ScalarType::Byte, device);
        shape.back() = k / kBlock;
        scale_rows = scales = empty(shape, ScalarType::Byte, device);
    }
    check_code(kmcts_mxfp4_quantize(flat.const_data_ptr(), element_code(x.scalar_type()), ldx, code_rows.mutable_data_ptr(),
                                    strides.codes, scale_rows.mutable_data_ptr(), strides.scales, rows, i32(k),
                                    current_stream(device)),
               "kmcts_mxfp4_quantize");
    if (out_codes) mark_written(codes), mark_written(scales);
    return {codes, scales};
}

Tensor mxfp4_dequantize(const Tensor& codes, const Tensor& scales, const std::optional<Tensor>& out,
                        const std::optional<ScalarType>& dtype) {
    const int device = cuda_index(codes);
    if (scales.dim() != codes.dim() || scales.sizes().slice(0, scales.dim() - (scales.dim() > 0)) !=
                                           codes.sizes().slice(0, codes.dim() - (codes.dim() > 0)))
        throw py::value_error(text("q scales must go with codes of shape ", shape_text(codes.sizes()), ", got ",
                                   shape_text(scales.sizes())));
    const Tensor code_rows = as_rows("q codes", codes), scale_rows = as_rows("q scales", scales);
    const PairStrides strides = check_pair("q", code_rows, scale_rows, 2, device);
    const int64_t rows = code_rows.size(0), k = 2 * code_rows.size(1);
    check_sizes({k});
    const ScalarType type = dtype ? *dtype : out ? out->scalar_type() : ScalarType::BFloat16;
    if (type != ScalarType::BFloat16 && type != ScalarType::Half && type != ScalarType::Float)
        throw py::type_error(text("values must be bfloat16, float16 or float32, got ", type_name(type)));
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    c10::SmallVector<int64_t, 5> shape(codes.sizes().begin(), codes.sizes().end());
    shape.back() = k;
    Tensor values, value_rows;
    int64_t ldo = k;
    if (out) {
        values = *out;
        check_writable("out", values);
        check_shape("out", values, shape);
        value_rows = as_rows("out", values);
        ldo = check_rows("out", value_rows, 2, {type}, device, kBlock);
    } else {
        value_rows = values = empty(shape, type, device);
    }
    check_code(kmcts_mxfp4_dequantize(code_rows.const_data_ptr(), strides.codes, scale_rows.const_data_ptr(), strides.scales,
                                      value_rows.mutable_data_ptr(), element_code(type), ldo, rows, i32(k),
                                      current_stream(device)),
               "kmcts_mxfp4_dequantize");
    if (out) mark_written(values);
    return values;
}

Tensor mxfp4_gemm(const Tensor& a, const Tensor& a_scales, const Tensor& b, const Tensor& b_scales,
                  const std::optional<Tensor>& ends, const std::optional<Tensor>& out, int kernel,
                  const std::optional<Tensor>& status) {
    const int device = cuda_index(a);
    const PairStrides lda = check_pair("a", a, a_scales, 2, device);
    const PairStrides ldb = check_pair("b", b, b_scales, ends ? 3 : 2, device);
    const int64_t rows = a.size(0), k = 2 * a.size(1), n = b.size(-2);
    if (b.size(-1) != a.size(1))
        throw py::value_error(text("inner dimensions differ: a has K=", k, ", b has K=", 2 * b.size(-1)));
    check_sizes({rows, n, k});
    int groups = 1;
    if (ends) {
        groups = check_groups(*ends, device);
        if (b.size(0) != groups) throw py::value_error(text("b holds ", b.size(0), " groups, ends ", groups));
    }
    int* const status_ptr = status_pointer(status, device);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    Tensor y;
    int64_t ldy = n;
    if (out) {
        y = *out;
        check_writable("out", y);
        ldy = check_rows("out", y, 2, {ScalarType::BFloat16}, device, 8);
        check_shape("out", y, {rows, n});
    } else {
        y = empty({rows, n}, ScalarType::BFloat16, device);
    }
    check_code(kmcts_mxfp4_gemm(a.const_data_ptr(), lda.codes, a_scales.const_data_ptr(), lda.scales, b.const_data_ptr(),
                                groups > 1 ? b.stride(0) : 0, ldb.codes, b_scales.const_data_ptr(),
                                groups > 1 ? b_scales.stride(0) : 0, ldb.scales, y.mutable_data_ptr(), ldy,
                                ends ? ends->const_data_ptr<int>() : nullptr, groups, i32(rows), i32(n), i32(k),
                                out ? 0 : KMCTS_GROUPED_ZERO_REST, kernel, current_stream(device), status_ptr),
               "kmcts_mxfp4_gemm");
    if (out) mark_written(y);
    return y;
}

}  // namespace

PYBIND11_MODULE(kmcts_torch_calls, m) {
    m.doc() = "Expert-layer calls on torch tensors (see kernel_mcts_b200.grouped and kernel_mcts_b200.mxfp4).";
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& failure) {
            const py::object error = py::module_::import("kernel_mcts_b200._native").attr("KmctsError");
            PyErr_SetObject(error.ptr(), error(failure.code, failure.call).ptr());
        }
    });
    // A launch waits while the device's queue is full: other threads go on meanwhile.
    const py::call_guard<py::gil_scoped_release> unlocked;
    m.def("grouped_gemm", &grouped_gemm, unlocked);
    m.def("grouped_gemm_wgrad", &grouped_gemm_wgrad, unlocked);
    m.def("grouped_linear", &grouped_linear, unlocked);
    m.def("mxfp4_quantize", &mxfp4_quantize, unlocked);
    m.def("mxfp4_dequantize", &mxfp4_dequantize, unlocked);
    m.def("mxfp4_gemm", &mxfp4_gemm, unlocked);
}
