// Host path of the operators whose calls are short: the 8-bit checkpoints (SwiGLU, RMSNorm, the pair) and the router's balance
// loss, as C++ autograd functions over the library's own C entry points.  The backward of a Python autograd function runs in the engine's
// device thread and has to take the interpreter's lock there, on a core whose caches are cold: forward + backward of a SwiGLU of
// 64 x 4096 bf16 in a loop take 107 us that way and 58 here, where those of a view, which launch nothing, take 32 (on an
// emptier host 46, 31 and 17).
//
// Eager GPU tensors come here (cute_kernels/_native.py); while a graph is traced the Python autograd functions with their
// `cute::` custom ops are taken instead.  Same kernels, same buffers, same results.
//
// Nothing here is linked against the kernel library: `load` opens it by the path the package uses and looks the entry
// points up, so that another build of it can be put in place.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include "../../include/cute_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
#define CK_ENTRY(name) decltype(&::name) name = nullptr
    CK_ENTRY(ck_status_string);
    CK_ENTRY(ck_abi_version);
    CK_ENTRY(ck_mx8_quantize);
    CK_ENTRY(ck_mx8_dequantize);
    CK_ENTRY(ck_swiglu_forward_mx8);
    CK_ENTRY(ck_swiglu_backward_mx8);
    CK_ENTRY(ck_rmsnorm_forward_mx8);
    CK_ENTRY(ck_rmsnorm_backward_mx8_workspace_size);
    CK_ENTRY(ck_rmsnorm_backward_mx8);
    CK_ENTRY(ck_moe_balance_loss_workspace_size);
    CK_ENTRY(ck_moe_balance_loss_forward);
    CK_ENTRY(ck_moe_balance_loss_backward);
#undef CK_ENTRY
} lib;

template <typename F>
void look_up(void* handle, const char* name, F& f) {
    f = reinterpret_cast<F>(dlsym(handle, name));
    TORCH_CHECK(f != nullptr, "the kernel library has no ", name, ": rebuild it");
}

void load(const std::string& path, int abi_version) {
    void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(handle != nullptr, "cannot open ", path, ": ", dlerror());
#define CK_ENTRY(name) look_up(handle, #name, lib.name)
    CK_ENTRY(ck_status_string);
    CK_ENTRY(ck_abi_version);
    CK_ENTRY(ck_mx8_quantize);
    CK_ENTRY(ck_mx8_dequantize);
    CK_ENTRY(ck_swiglu_forward_mx8);
    CK_ENTRY(ck_swiglu_backward_mx8);
    CK_ENTRY(ck_rmsnorm_forward_mx8);
    CK_ENTRY(ck_rmsnorm_backward_mx8_workspace_size);
    CK_ENTRY(ck_rmsnorm_backward_mx8);
    CK_ENTRY(ck_moe_balance_loss_workspace_size);
    CK_ENTRY(ck_moe_balance_loss_forward);
    CK_ENTRY(ck_moe_balance_loss_backward);
#undef CK_ENTRY
    TORCH_CHECK(lib.ck_abi_version() == abi_version, "libcute_hip.so has ABI version ", lib.ck_abi_version(),
                ", this package needs ", abi_version, ": rebuild it");
}

// ---- operands ------------------------------------------------------------------------------------------------------
void check(int status, const char* name) {
    TORCH_CHECK(status == CK_OK, name, " failed: ", lib.ck_status_string(status), " (status ", status, ")");
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return CK_F32;
        case at::kHalf: return CK_F16;
        case at::kBFloat16: return CK_BF16;
        default:
            TORCH_CHECK_VALUE(false, "unsupported dtype (", t, "); the HIP kernels take float32, float16 and bfloat16");
    }
}

// `others` are on the first operand's GPU, of its dtype and (unless `shapes` is false) its shape
void alike(const char* what, const Tensor& first, std::initializer_list<const Tensor*> others, bool shapes = true) {
    TORCH_CHECK(first.is_cuda(), "cute_kernels HIP kernels need GPU tensors; got a tensor on ", first.device());
    for (const Tensor* t : others) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->device() == first.device(), "tensors on different devices (", first.device(), " and ", t->device(), ")");
        TORCH_CHECK_VALUE(t->scalar_type() == first.scalar_type(), what, ": expected ", first.scalar_type(), ", got ",
                          t->scalar_type());
        TORCH_CHECK_VALUE(!shapes || t->sizes() == first.sizes(), what, ": operands of shapes ", first.sizes(), " and ", t->sizes());
    }
}

struct Rows {
    int64_t count, H;
};
Rows rows_of(const Tensor& t) {
    TORCH_CHECK_VALUE(t.dim() >= 1, "a tensor with rows is needed, got a scalar");
    const int64_t H = t.size(-1);
    return {H > 0 ? t.numel() / H : 0, H};
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) {  // (call it with the tensor's device current)
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// what an operator keeps: codes, scale bytes, 1 / rms - the layout of mx8_kept_offsets in cute_kernels/_C.py
struct Kept {
    int64_t scales, rstd, total;
    Kept(int64_t rows, int64_t H, bool with_rstd) {
        scales = (rows * H + 15) & -16;
        const int64_t end = scales + rows * ((H + 31) / 32);
        rstd = with_rstd ? (end + 15) & -16 : end;
        total = with_rstd ? rstd + 4 * rows : end;
    }
};
Tensor bytes(int64_t n, const Tensor& like, at::ScalarType type = at::kChar) {
    return at::empty({n}, like.options().dtype(type));
}

// Gradients the kernels computed know nothing of how they depend on what they came from: where a graph of the backward is
// asked for (create_graph=True), going through them is an error instead of a gradient with a part missing.
// (The error stands between the gradients and the operator's own inputs, so that it is met on every way to them.)
variable_list not_differentiable(variable_list grads) {
    const auto node = at::GradMode::is_enabled() ? torch::autograd::get_current_node() : nullptr;
    if (node == nullptr) return grads;
    const auto error = std::make_shared<torch::autograd::Error>(
        "cute_kernels: the backward of this operator has no derivative of its own", torch::autograd::edge_list(node->next_edges()));
    for (Tensor& g : grads) {
        if (!g.defined()) continue;
        g = g.detach();
        torch::autograd::set_history(g, error);
    }
    return grads;
}

// ---- the pair --------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> mx8_quantize(const Tensor& input) {
    at::NoGradGuard no_grad;
    alike("mx8_quantize", input, {});
    const Tensor x = input.contiguous();
    const Rows r = rows_of(x);
    const c10::DeviceGuard guard(x.device());
    auto shape = x.sizes().vec();
    Tensor codes = at::empty(shape, x.options().dtype(at::kChar));
    shape.back() = (r.H + 31) / 32;
    Tensor scales = at::empty(shape, x.options().dtype(at::kByte));
    check(lib.ck_mx8_quantize(data(x), data(codes), data(scales), r.count, r.H, dtype_code(x.scalar_type()), stream_of(x)),
          "ck_mx8_quantize");
    return {codes, scales};
}

Tensor mx8_dequantize(const Tensor& input_codes, const Tensor& input_scales, at::ScalarType dtype) {
    at::NoGradGuard no_grad;
    TORCH_CHECK(input_codes.is_cuda(), "cute_kernels HIP kernels need GPU tensors; got a tensor on ", input_codes.device());
    TORCH_CHECK(input_scales.device() == input_codes.device(), "tensors on different devices (", input_codes.device(), " and ",
                input_scales.device(), ")");
    TORCH_CHECK_VALUE(input_codes.scalar_type() == at::kChar && input_scales.scalar_type() == at::kByte,
                      "mx8_dequantize: codes are int8 and scales uint8, got ", input_codes.scalar_type(), " and ",
                      input_scales.scalar_type());
    const Tensor codes = input_codes.contiguous(), scales = input_scales.contiguous();
    const Rows r = rows_of(codes);
    auto shape = codes.sizes().vec();
    shape.back() = (r.H + 31) / 32;
    TORCH_CHECK_VALUE(scales.sizes() == at::IntArrayRef(shape), "mx8_dequantize: scales ", scales.sizes(),
                      " do not go with codes ", codes.sizes(), ": one per 32 elements of a row");
    const int code = dtype_code(dtype);
    const c10::DeviceGuard guard(codes.device());
    Tensor output = at::empty(codes.sizes(), codes.options().dtype(dtype));
    check(lib.ck_mx8_dequantize(data(codes), data(scales), data(output), r.count, r.H, code, stream_of(codes)),
          "ck_mx8_dequantize");
    return output;
}

// ---- SwiGLU -----------------------------------------------------------------------------------------------------------
struct SwigluMX8 : torch::autograd::Function<SwigluMX8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& gate_in, const Tensor& up_in) {
        alike("swiglu", gate_in, {&up_in});
        const Tensor gate = gate_in.contiguous(), up = up_in.contiguous();
        const Rows r = rows_of(gate);
        const c10::DeviceGuard guard(gate.device());
        Tensor output = at::empty(gate.sizes(), gate.options());
        const Kept k(2 * r.count, r.H, false);
        Tensor kept = bytes(k.total, gate);
        if (r.count > 0) {
            char *c = (char*)data(kept), *s = c + k.scales;
            const int64_t blocks = (r.H + 31) / 32;
            check(lib.ck_swiglu_forward_mx8(data(gate), data(up), r.H, data(output), c, c + r.count * r.H, r.H, s,
                                            s + r.count * blocks, blocks, r.count, r.H, dtype_code(gate.scalar_type()),
                                            stream_of(gate)),
                  "ck_swiglu_forward_mx8");
        }
        ctx->save_for_backward({kept});
        return output;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor dy = grads[0].contiguous(), kept = ctx->get_saved_variables()[0];
        const Rows r = rows_of(dy);
        const c10::DeviceGuard guard(dy.device());
        Tensor gate_grad = at::empty(dy.sizes(), dy.options()), up_grad = at::empty(dy.sizes(), dy.options());
        if (r.count > 0) {
            const Kept k(2 * r.count, r.H, false);
            const char *c = (const char*)data(kept), *s = c + k.scales;
            const int64_t blocks = (r.H + 31) / 32;
            check(lib.ck_swiglu_backward_mx8(c, c + r.count * r.H, r.H, s, s + r.count * blocks, blocks, data(dy),
                                             data(gate_grad), data(up_grad), r.H, nullptr, r.count, r.H,
                                             dtype_code(dy.scalar_type()), stream_of(dy)),
                  "ck_swiglu_backward_mx8");
        }
        return not_differentiable({gate_grad, up_grad});
    }
};

// x [..., 2 H] = (up | gate)
struct SwigluUnchunkedMX8 : torch::autograd::Function<SwigluUnchunkedMX8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_in) {
        alike("swiglu_unchunked", x_in, {});
        const Tensor x = x_in.contiguous();
        auto shape = x.sizes().vec();
        TORCH_CHECK_VALUE(!shape.empty() && shape.back() % 2 == 0, "last dimension of x must be even");
        const int64_t H = shape.back() / 2, rows = H > 0 ? x.numel() / (2 * H) : 0;
        shape.back() = H;
        const c10::DeviceGuard guard(x.device());
        Tensor output = at::empty(shape, x.options());
        const Kept k(2 * rows, H, false);
        Tensor kept = bytes(k.total, x);
        if (rows > 0) {
            char *c = (char*)data(kept), *s = c + k.scales, *up = (char*)data(x);
            const int64_t blocks = (H + 31) / 32;
            check(lib.ck_swiglu_forward_mx8(up + H * x.element_size(), up, 2 * H, data(output), c + H, c, 2 * H, s + blocks, s,
                                            2 * blocks, rows, H, dtype_code(x.scalar_type()), stream_of(x)),
                  "ck_swiglu_forward_mx8");
        }
        ctx->save_for_backward({kept});
        return output;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor dy = grads[0].contiguous(), kept = ctx->get_saved_variables()[0];
        const Rows r = rows_of(dy);
        auto shape = dy.sizes().vec();
        shape.back() = 2 * r.H;
        const c10::DeviceGuard guard(dy.device());
        Tensor x_grad = at::empty(shape, dy.options());
        if (r.count > 0) {
            const Kept k(2 * r.count, r.H, false);
            const char *c = (const char*)data(kept), *s = c + k.scales;
            char* up = (char*)data(x_grad);
            const int64_t blocks = (r.H + 31) / 32;
            check(lib.ck_swiglu_backward_mx8(c + r.H, c, 2 * r.H, s + blocks, s, 2 * blocks, data(dy),
                                             up + r.H * dy.element_size(), up, 2 * r.H, nullptr, r.count, r.H,
                                             dtype_code(dy.scalar_type()), stream_of(dy)),
                  "ck_swiglu_backward_mx8");
        }
        return not_differentiable({x_grad});
    }
};

// ---- RMSNorm ------------------------------------------------------------------------------------------------------------
Tensor contiguous_or_none(const std::optional<Tensor>& t) { return t.has_value() && t->defined() ? t->contiguous() : Tensor(); }

// output, the sum (undefined without a residual), what is kept
std::tuple<Tensor, Tensor, Tensor> rmsnorm_forward(const char* what, const Tensor& x, const Tensor& residual,
                                                   const Tensor& weight, double eps) {
    alike(what, x, {&residual});
    alike(what, x, {&weight}, false);
    const Rows r = rows_of(x);
    TORCH_CHECK_VALUE(!weight.defined() || (weight.dim() == 1 && weight.numel() == r.H), what, ": weight of shape ",
                      weight.defined() ? weight.sizes() : at::IntArrayRef(), " for rows of ", r.H);
    Tensor output = at::empty(x.sizes(), x.options()), sum;
    if (residual.defined()) sum = at::empty(x.sizes(), x.options());
    const Kept k(r.count, r.H, true);
    Tensor kept = bytes(k.total, x);
    if (r.count > 0) {
        char* c = (char*)data(kept);
        check(lib.ck_rmsnorm_forward_mx8(data(x), data(residual), data(weight), data(output), data(sum), c, c + k.scales,
                                         (float*)(c + k.rstd), r.count, r.H, (float)eps, dtype_code(x.scalar_type()),
                                         stream_of(x)),
              "ck_rmsnorm_forward_mx8");
    }
    return {output, sum, kept};
}

// gradient of the normalised rows (plus sum_grad where defined) and of the weight
std::tuple<Tensor, Tensor> rmsnorm_backward(const Tensor& kept, const Tensor& weight, const Tensor& dy, const Tensor& sum_grad) {
    const Rows r = rows_of(dy);
    const Kept k(r.count, r.H, true);
    const int dtype = dtype_code(dy.scalar_type());
    Tensor x_grad = at::empty(dy.sizes(), dy.options()), weight_grad, workspace;
    int64_t nbytes = 0;
    if (weight.defined()) {
        weight_grad = at::empty(weight.sizes(), weight.options());
        nbytes = std::max<int64_t>(lib.ck_rmsnorm_backward_mx8_workspace_size(r.count, r.H, dtype), 16);
        workspace = bytes(nbytes, dy, at::kByte);
    }
    const char* c = (const char*)data(kept);
    check(lib.ck_rmsnorm_backward_mx8(c, c + k.scales, data(weight), data(dy), (const float*)(c + k.rstd), data(sum_grad),
                                      data(x_grad), data(weight_grad), data(workspace), nbytes, r.count, r.H, dtype,
                                      stream_of(dy)),
          "ck_rmsnorm_backward_mx8");
    return {x_grad, weight_grad};
}

struct RMSNormMX8 : torch::autograd::Function<RMSNormMX8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_in, double eps) {
        const c10::DeviceGuard guard(x.device());
        const Tensor weight = contiguous_or_none(weight_in);
        auto [output, sum, kept] = rmsnorm_forward("rmsnorm", x.contiguous(), Tensor(), weight, eps);
        ctx->save_for_backward({kept, weight});
        return output;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(grads[0].device());
        auto [x_grad, weight_grad] = rmsnorm_backward(saved[0], saved[1], grads[0].contiguous(), Tensor());
        return not_differentiable({x_grad, weight_grad, Tensor()});
    }
};

struct ResidualRMSNormMX8 : torch::autograd::Function<ResidualRMSNormMX8> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual,
                                 const std::optional<Tensor>& weight_in, double eps) {
        const c10::DeviceGuard guard(x.device());
        const Tensor weight = contiguous_or_none(weight_in);
        auto [output, sum, kept] = rmsnorm_forward("residual rmsnorm", x.contiguous(), residual.contiguous(), weight, eps);
        ctx->save_for_backward({kept, weight});
        ctx->set_materialize_grads(false);
        return {output, sum};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor& weight = saved[1];
        if (!grads[0].defined()) {
            // only the sum was used: the normalisation has no gradient
            return {grads[1], grads[1], weight.defined() ? at::zeros_like(weight) : Tensor(), Tensor()};
        }
        const c10::DeviceGuard guard(grads[0].device());
        auto [x_grad, weight_grad] = rmsnorm_backward(saved[0], weight, grads[0].contiguous(),
                                                      grads[1].defined() ? grads[1].contiguous() : Tensor());
        // the sum hands the same gradient to both of its terms
        return not_differentiable({x_grad, x_grad, weight_grad, Tensor()});
    }
};

// ---- balance loss ---------------------------------------------------------------------------------------------------------
// distance of the rows of a [T, E] matrix with unit column stride
int64_t row_distance(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& selected,
                                 const std::optional<Tensor>& mask_in) {
        const Tensor mask = contiguous_or_none(mask_in);
        TORCH_CHECK(logits.is_cuda(), "cute_kernels HIP kernels need GPU tensors; got a tensor on ", logits.device());
        for (const Tensor* t : {&selected, &mask})
            TORCH_CHECK(!t->defined() || t->device() == logits.device(), "tensors on different devices (", logits.device(),
                        " and ", t->device(), ")");
        TORCH_CHECK_VALUE(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
                          "moe_balance_loss: logits need unit stride over the experts");
        const int64_t T = logits.size(0), E = logits.size(1);
        TORCH_CHECK_VALUE(selected.scalar_type() == at::kLong && selected.dim() == 2 && selected.size(0) == T &&
                              selected.is_contiguous(),
                          "moe_balance_loss: selected must be dense int64 [tokens, k]");
        TORCH_CHECK_VALUE(!mask.defined() || (mask.scalar_type() == at::kBool && mask.numel() == T),
                          "moe_balance_loss: the mask is one bool per token");
        const int dtype = dtype_code(logits.scalar_type());
        const c10::DeviceGuard guard(logits.device());
        const auto f32 = logits.options().dtype(at::kFloat);
        Tensor balance = at::empty({}, f32), z = at::empty({}, f32), shares = at::empty({E + 1}, f32);
        Tensor counts = at::empty({E}, logits.options().dtype(at::kInt)), workspace;
        const int64_t nbytes = lib.ck_moe_balance_loss_workspace_size(T, E);
        if (nbytes > 0) workspace = bytes(nbytes, logits, at::kByte);
        check(lib.ck_moe_balance_loss_forward(data(logits), row_distance(logits), selected.data_ptr<int64_t>(), data(mask),
                                              balance.data_ptr<float>(), z.data_ptr<float>(), counts.data_ptr<int>(),
                                              shares.data_ptr<float>(), data(workspace), nbytes, T, E, selected.size(1), dtype,
                                              stream_of(logits)),
              "ck_moe_balance_loss_forward");
        ctx->save_for_backward({logits, mask, shares});
        ctx->mark_non_differentiable({counts});
        ctx->set_materialize_grads(false);
        return {balance, z, counts};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &mask = saved[1], &shares = saved[2];
        const c10::DeviceGuard guard(logits.device());
        Tensor d_logits = at::empty(logits.sizes(), logits.options());
        check(lib.ck_moe_balance_loss_backward(data(logits), row_distance(logits), data(mask), shares.data_ptr<float>(),
                                               (const float*)data(grads[0]), (const float*)data(grads[1]), data(d_logits),
                                               logits.size(0), logits.size(1), dtype_code(logits.scalar_type()),
                                               stream_of(logits)),
              "ck_moe_balance_loss_backward");
        return not_differentiable({d_logits, Tensor(), Tensor()});
    }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    const auto unlocked = py::call_guard<py::gil_scoped_release>();
    // the signatures this module was compiled with: `load` casts the library's entry points to them
    m.attr("abi_version") = CK_ABI_VERSION;
    m.def("load", &load);
    m.def("not_differentiable", [](const std::vector<std::optional<Tensor>>& grads) {
        variable_list given;
        for (const auto& g : grads) given.push_back(g.value_or(Tensor()));
        std::vector<std::optional<Tensor>> out;
        for (const Tensor& g : not_differentiable(given)) out.push_back(g.defined() ? std::optional<Tensor>(g) : std::nullopt);
        return out;
    });
    m.def("mx8_quantize", &mx8_quantize, unlocked);
    m.def("mx8_dequantize", &mx8_dequantize, unlocked);
    m.def("swiglu", [](const Tensor& gate, const Tensor& up) { return SwigluMX8::apply(gate, up); }, unlocked);
    m.def("swiglu_unchunked", [](const Tensor& x) { return SwigluUnchunkedMX8::apply(x); }, unlocked);
    m.def("rmsnorm",
          [](const Tensor& x, const std::optional<Tensor>& weight, double eps) { return RMSNormMX8::apply(x, weight, eps); },
          unlocked);
    m.def("residual_rmsnorm",
          [](const Tensor& x, const Tensor& residual, const std::optional<Tensor>& weight, double eps) {
              const auto out = ResidualRMSNormMX8::apply(x, residual, weight, eps);
              return std::make_tuple(out[0], out[1]);
          },
          unlocked);
    m.def("moe_balance_loss",
          [](const Tensor& logits, const Tensor& selected, const std::optional<Tensor>& mask) {
              const auto out = BalanceLoss::apply(logits, selected, mask);
              return std::make_tuple(out[0], out[1], out[2]);
          },
          unlocked);
}
