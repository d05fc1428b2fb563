// tcg_torch.cpp -- the torch binding of the calls that are bound by the host
// when they are small: int8 and grouped products of a few rows, and the
// differentiable layers.  Checks, results and launches of a call are made here
// in one go (a layer's training step of 515 x 1024 x 768 took 120 us from
// Python, where the autograd engine alone takes 50); the arithmetic is
// libtcgemm.so's, through its C ABI.  Results, checks and messages are those
// of rows.py, which documents them.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/torch.h>

#include <optional>

#include "../../include/tcgemm.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// A status of the C ABI on its way to Python, where it becomes a TcgError.
struct StatusError : std::runtime_error {
    StatusError(const char* function, tcg_status s)
        : std::runtime_error(std::string(function) + ": status " + std::to_string(static_cast<int>(s)) + " (" +
                             tcg_status_string(s) + ")"),
          fn(function),
          status(s)
    {
    }
    std::string fn;
    tcg_status status;
};

void check_status(const char* fn, tcg_status s)
{
    if (s != TCG_SUCCESS) throw StatusError(fn, s);
}

// One launch's device and stream: those of the tensor it works on.
struct On {
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
    c10::cuda::CUDAGuard guard;
    void* stream;
};

bool is_half(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
bool is_type(at::ScalarType t) { return t == at::kFloat || is_half(t); }
tcg_dtype type_of(at::ScalarType t) { return t == at::kFloat ? TCG_F32 : (t == at::kHalf ? TCG_F16 : TCG_BF16); }

int narrow(int64_t n, const char* what)
{
    TORCH_CHECK(n >= 0 && n <= INT_MAX, what, " is too large");
    return static_cast<int>(n);
}

void same_device(const Tensor& like, const char* name, const Tensor& t)
{
    TORCH_CHECK(t.get_device() == like.get_device(), name, " must be on the same device as the other operands");
}

void check_offsets(const Tensor& offsets, int64_t groups, const Tensor& like)
{
    TORCH_CHECK(offsets.is_cuda() && offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.is_contiguous(),
                "offsets must be a contiguous 1-D CUDA int32 tensor");
    TORCH_CHECK(offsets.numel() == groups + 1, "offsets must have one entry more than there are groups");
    TORCH_CHECK(groups > 0 && groups <= TCG_MAX_GROUPS, "the number of groups must be 1 to ", TCG_MAX_GROUPS);
    same_device(like, "offsets", offsets);
}

void check_floats(const char* name, const Tensor& t, at::IntArrayRef shape, const Tensor& like)
{
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous(), name,
                " must be a contiguous CUDA float32 tensor");
    TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape);
    same_device(like, name, t);
}

const int32_t* offsets_ptr(const Tensor& o) { return o.defined() ? o.const_data_ptr<int32_t>() : nullptr; }

// x's shape with another last extent
Tensor like_rows(const Tensor& x, int64_t last, at::ScalarType type)
{
    at::DimVector shape(x.sizes());
    shape.back() = last;
    return at::empty(shape, x.options().dtype(type));
}

int64_t rows_of(const Tensor& x) { return x.size(-1) ? x.numel() / x.size(-1) : 0; }

bool overlap(const Tensor& a, const Tensor& b)
{
    const char *pa = static_cast<const char*>(a.const_data_ptr()), *pb = static_cast<const char*>(b.const_data_ptr());
    return pa < pb + b.nbytes() && pb < pa + a.nbytes();
}

// The given result, or a new one, whose rows outside the groups become zeros.
Tensor grouped_out(const OptTensor& out, const Tensor& A, std::initializer_list<OptTensor> inputs, int64_t N,
                   at::ScalarType type, int* zero_rest)
{
    *zero_rest = !out.has_value();
    if (!out) return at::empty({A.size(0), N}, A.options().dtype(type));
    TORCH_CHECK(out->is_cuda() && out->is_contiguous() && out->dim() == 2 && out->size(0) == A.size(0) &&
                    out->size(1) == N && out->scalar_type() == type,
                "out must be a contiguous CUDA tensor of shape [", A.size(0), ", ", N, "] and type ", type);
    same_device(A, "out", *out);
    for (const OptTensor& t : inputs) TORCH_CHECK(!t || !overlap(*out, *t), "out must not overlap the inputs");
    TORCH_CHECK(!(at::GradMode::is_enabled() && out->requires_grad()), "out must not require grad");
    out->unsafeGetTensorImpl()->bump_version();  // autograd: what was saved of it is stale
    return *out;
}

// ------------------------------------------------------- products, checked --

void product(const Tensor& A, const Tensor& B, const Tensor& offsets, bool nk, const Tensor& C, int zero_rest)
{
    const On on(A);
    check_status("tcg_gemm_16_grouped",
                 tcg_gemm_16_grouped(A.const_data_ptr(), B.const_data_ptr(), type_of(A.scalar_type()),
                                     C.mutable_data_ptr(), type_of(C.scalar_type()), offsets_ptr(offsets),
                                     B.dim() == 3 ? narrow(B.size(0), "the number of groups") : 1,
                                     narrow(rows_of(A), "the number of rows"), narrow(C.size(-1), "N"),
                                     narrow(A.size(-1), "K"), nk ? TCG_B_NK : TCG_B_KN, zero_rest, on.stream));
}

std::pair<Tensor, Tensor> quantize(const Tensor& x)
{
    Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
    Tensor scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    const On on(x);
    check_status("tcg_quantize_rows_s8",
                 tcg_quantize_rows_s8(x.const_data_ptr(), type_of(x.scalar_type()),
                                      static_cast<int8_t*>(codes.mutable_data_ptr()),
                                      static_cast<float*>(scales.mutable_data_ptr()), scales.numel(),
                                      narrow(x.size(-1), "K"), on.stream));
    return {codes, scales};
}

Tensor dequantize(const Tensor& codes, const Tensor& scales, at::ScalarType type)
{
    Tensor out = at::empty(codes.sizes(), codes.options().dtype(type));
    const On on(codes);
    check_status("tcg_dequantize_rows_s8",
                 tcg_dequantize_rows_s8(static_cast<const int8_t*>(codes.const_data_ptr()),
                                        static_cast<const float*>(scales.const_data_ptr()), out.mutable_data_ptr(),
                                        type_of(type), scales.numel(), narrow(codes.size(-1), "K"), on.stream));
    return out;
}

// dW[groups, N, K] (2-D without groups)
Tensor weight_gradient(const Tensor& dy, const Tensor& x, const Tensor& offsets)
{
    const int64_t N = dy.size(-1), K = x.size(-1);
    const int groups = offsets.defined() ? narrow(offsets.numel() - 1, "the number of groups") : 1;
    Tensor dW = offsets.defined() ? at::empty({groups, N, K}, dy.options()) : at::empty({N, K}, dy.options());
    const On on(dy);
    check_status("tcg_gemm_16_grouped_wgrad",
                 tcg_gemm_16_grouped_wgrad(dy.const_data_ptr(), x.const_data_ptr(), type_of(dy.scalar_type()),
                                           dW.mutable_data_ptr(), type_of(dy.scalar_type()), offsets_ptr(offsets),
                                           groups, narrow(rows_of(dy), "the number of rows"), narrow(N, "N"),
                                           narrow(K, "K"), on.stream));
    return dW;
}

// ------------------------------------------------------------------ entries --

std::pair<Tensor, Tensor> quantize_rows(const Tensor& x)
{
    TORCH_CHECK(x.is_cuda() && is_type(x.scalar_type()) && x.is_contiguous() && x.dim() >= 1,
                "x must be a contiguous CUDA float32, float16 or bfloat16 tensor with at least one axis");
    at::NoGradGuard no_grad;
    return quantize(x);
}

Tensor linear_int8(const Tensor& x, const Tensor& BT, const OptTensor& offsets, const Tensor& scale_b,
                   const OptTensor& bias, const OptTensor& out)
{
    TORCH_CHECK(x.is_cuda() && BT.is_cuda(), "x and BT must be CUDA tensors");
    TORCH_CHECK(offsets ? x.dim() == 2 && BT.dim() == 3 : x.dim() >= 1 && BT.dim() == 2,
                offsets ? "x must be 2-D and BT 3-D" : "BT must be 2-D");
    TORCH_CHECK(is_type(x.scalar_type()), "x must be float32, float16 or bfloat16");
    TORCH_CHECK(BT.scalar_type() == at::kChar, "BT must be int8");
    const int64_t N = BT.size(-2), K = BT.size(-1);
    TORCH_CHECK(x.size(-1) == K, "x cols must equal BT cols (both = K)");
    TORCH_CHECK(x.is_contiguous() && BT.is_contiguous(), "x and BT must be contiguous");
    TORCH_CHECK(K > 0, "K must not be 0");
    same_device(x, "BT", BT);
    const int groups = offsets ? narrow(BT.size(0), "the number of groups") : 1;
    if (offsets) check_offsets(*offsets, groups, x);
    const at::IntArrayRef channels = BT.sizes().slice(0, BT.dim() - 1);
    check_floats("scale_b", scale_b, channels, x);
    if (bias) check_floats("bias", *bias, channels, x);
    const int M = narrow(rows_of(x), "the number of rows");
    int zero_rest = 0;
    Tensor C = offsets ? grouped_out(out, x, {x, BT, offsets, scale_b, bias}, N, x.scalar_type(), &zero_rest) : like_rows(x, N, x.scalar_type());
    if (C.numel() == 0) return C;
    const On on(x);
    const auto call = [&](void* workspace, size_t bytes) {
        return tcg_linear_s8_grouped(
            x.const_data_ptr(), type_of(x.scalar_type()), static_cast<const int8_t*>(BT.const_data_ptr()),
            C.mutable_data_ptr(), type_of(x.scalar_type()), offsets ? offsets_ptr(*offsets) : nullptr, groups, M,
            narrow(N, "N"), narrow(K, "K"), static_cast<const float*>(scale_b.const_data_ptr()),
            bias ? static_cast<const float*>(bias->const_data_ptr()) : nullptr, zero_rest, workspace, bytes, on.stream);
    };
    // few rows usually need no workspace; the call says so before it launches anything
    tcg_status s = offsets || M > 4 ? TCG_ERR_WORKSPACE : call(nullptr, 0);
    if (s == TCG_ERR_WORKSPACE) {
        const size_t need = tcg_linear_s8_workspace_size(M, static_cast<int>(K));
        Tensor ws = at::empty({static_cast<int64_t>(need)}, x.options().dtype(at::kByte));
        s = call(ws.mutable_data_ptr(), need);
    }
    check_status("tcg_linear_s8_grouped", s);
    return C;
}

Tensor gemm_grouped(const Tensor& A, const Tensor& B, const Tensor& offsets, bool nk,
                    const std::optional<at::ScalarType>& out_dtype, const OptTensor& out)
{
    TORCH_CHECK(A.is_cuda() && B.is_cuda(), "A and B must be CUDA tensors");
    TORCH_CHECK(is_half(A.scalar_type()) && B.scalar_type() == A.scalar_type(),
                "A and B must both be float16 or both bfloat16");
    TORCH_CHECK(A.dim() == 2 && B.dim() == 3, "A must be 2-D and B 3-D");
    TORCH_CHECK(A.size(1) == B.size(nk ? 2 : 1), "A cols must equal K of B");
    TORCH_CHECK(A.is_contiguous() && B.is_contiguous(), "A and B must be contiguous");
    const at::ScalarType type = out_dtype.value_or(A.scalar_type());
    TORCH_CHECK(is_type(type), "out_dtype must be float16, bfloat16 or float32");
    same_device(A, "B", B);
    check_offsets(offsets, B.size(0), A);
    int zero_rest;
    Tensor C = grouped_out(out, A, {A, B, offsets}, B.size(nk ? 1 : 2), type, &zero_rest);
    product(A, B, offsets, nk, C, zero_rest);
    return C;
}

// y = x W^T per group.  Backward: dx = dy W (the same product with W's other
// layout), dW = dy^T x from x or from its int8 codes and scales.  Those are
// widened to the layer's type first: the tensor cores take 16-bit operands, and
// code * scale has more bits than one holds.  That rounding is as large as the
// result's own (bf16: error of dW 0.0023 of its size against 0.0017 unrounded,
// fp16 0.00028 against 0.00021) and a fifth of the codes' error against
// x (0.008 and more); a second operand for the remainders would double the product.  What one
// input's gradient alone needs is kept only where that is asked for.
struct LinearFunction : public torch::autograd::Function<LinearFunction> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& W,
                          const OptTensor& offsets_or_none, bool eight)
    {
        const Tensor offsets = offsets_or_none.value_or(Tensor());
        Tensor y = like_rows(x, W.size(-2), x.scalar_type());
        product(x, W, offsets, true, y, 1);
        Tensor kept, scales;
        if (W.requires_grad()) {
            if (eight)
                std::tie(kept, scales) = quantize(x);
            else
                kept = x;
        }
        ctx->save_for_backward({kept, scales, x.requires_grad() ? W : Tensor(), offsets});
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads)
    {
        torch::autograd::variable_list out(4);
        if (!grads[0].defined()) return out;
        const bool again = at::GradMode::is_enabled();
        {
            at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const Tensor &kept = saved[0], &scales = saved[1], &W = saved[2], &offsets = saved[3];
            Tensor dy = grads[0].contiguous();
            // (a slice of a larger gradient may start anywhere)
            if (reinterpret_cast<uintptr_t>(dy.const_data_ptr()) % 16 != 0) dy = dy.clone();
            // inputs that this pass asks for: x is the function's first, W its second
            if (W.defined() && ctx->needs_input_grad(0)) {
                out[0] = like_rows(dy, W.size(-1), dy.scalar_type());
                product(dy, W, offsets, false, out[0], 1);
            }
            if (kept.defined() && ctx->needs_input_grad(1))
                out[1] = weight_gradient(dy, scales.defined() ? dequantize(kept, scales, dy.scalar_type()) : kept,
                                         offsets);
        }
        if (again) {
            // recorded for a second differentiation, which these products do not have
            torch::autograd::variable_list both;
            for (const Tensor& t : out)
                if (t.defined()) both.push_back(t.detach().requires_grad_(true));
            both = (*std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that can be differentiated once",
                static_cast<int64_t>(both.size())))(std::move(both));
            size_t i = 0;
            for (Tensor& t : out)
                if (t.defined()) t = both[i++];
        }
        return out;
    }
};

Tensor linear(const Tensor& x, const Tensor& W, const OptTensor& offsets, bool eight)
{
    TORCH_CHECK(offsets ? x.dim() == 2 && W.dim() == 3 : x.dim() >= 1 && W.dim() == 2,
                offsets ? "x must be 2-D and W 3-D" : "W must be 2-D");
    TORCH_CHECK(x.is_cuda() && W.is_cuda(), "x and W must be CUDA tensors");
    TORCH_CHECK(is_half(x.scalar_type()) && W.scalar_type() == x.scalar_type(),
                "x and W must both be float16 or both bfloat16");
    TORCH_CHECK(x.size(-1) == W.size(-1), "x cols must equal W cols (both = K)");
    TORCH_CHECK(x.is_contiguous() && W.is_contiguous(), "x and W must be contiguous");
    TORCH_CHECK(W.size(-1) % 8 == 0, "K must be a multiple of 8");
    TORCH_CHECK(W.size(-2) % 8 == 0, "N must be a multiple of 8");
    TORCH_CHECK(W.numel() > 0, "W must not be empty");
    same_device(x, "W", W);
    if (offsets) check_offsets(*offsets, W.size(0), x);
    if (at::GradMode::is_enabled() && (x.requires_grad() || W.requires_grad()))
        return LinearFunction::apply(x, W, offsets, eight);
    Tensor y = like_rows(x, W.size(-2), x.scalar_type());
    product(x, W, offsets.value_or(Tensor()), true, y, 1);
    return y;
}

}  // namespace

PYBIND11_MODULE(_tcg_torch, m)
{
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const StatusError& e) {
            try {
                py::object type = py::module_::import("tensorcoreptx_b200._native").attr("TcgError");
                py::object value = type(e.fn, static_cast<int>(e.status));
                PyErr_SetObject(type.ptr(), value.ptr());
            } catch (py::error_already_set& nested) {
                nested.restore();
            }
        }
    });
    m.def("quantize_rows", &quantize_rows);
    m.def("linear_int8", &linear_int8);
    m.def("gemm_grouped", &gemm_grouped);
    m.def("linear", &linear);
}
