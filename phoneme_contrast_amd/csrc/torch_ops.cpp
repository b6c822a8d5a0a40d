// torch operators over the C ABI, for calls that are shorter than their way through Python: torch.ops.pcx.layer_norm
// with its gradient (a Python autograd function costs 50 us of host time per training call at 24 x 128, where the
// kernels take 10).  Checks, allocation and the current stream as in phoneme_contrast_amd/layers.py's contract.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <tuple>

#include "pcx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The C entry points of the library that the process has loaded (linked here, libpcx.so could be a second copy and
// another build than the one that serves all other calls).
struct Entries {
    decltype(&pcx_last_error) last_error;
    decltype(&pcx_layernorm_workspace_bytes) workspace_bytes;
    decltype(&pcx_layernorm_forward) layernorm_forward;
    decltype(&pcx_layernorm_backward) layernorm_backward;
} pcx;

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PCX_F32;
        case at::kBFloat16: return PCX_BF16;
        case at::kHalf: return PCX_F16;
        default: return -1;
    }
}

void check_status(int rc, const char* what) {
    if (rc == PCX_OK) return;
    char msg[512];
    pcx.last_error(msg, sizeof msg);
    if (rc == PCX_EINVAL || rc == PCX_ESHAPE) TORCH_CHECK_VALUE(false, msg);
    TORCH_CHECK(false, what, " failed (", rc, "): ", msg);
}

// [..., D] as (tensor, rows, row stride): in place where the rows are evenly spaced with adjacent values, else a copy
std::tuple<Tensor, int64_t, int64_t> rows_of(const Tensor& t, int64_t D) {
    const int64_t rows = t.numel() / D;
    if (t.is_contiguous()) return {t, rows, D};
    // one trailing axis of adjacent values, and leading axes that step evenly (size-1 axes anywhere)
    int64_t inner = 1, k = t.dim() - 1;
    bool even = true;
    for (; k >= 0 && inner < D; --k) {
        even = even && (t.size(k) == 1 || t.stride(k) == inner);
        inner *= t.size(k);
    }
    int64_t step = -1, span = 0;
    for (; k >= 0 && even; --k) {
        if (t.size(k) == 1) continue;
        if (step < 0) step = t.stride(k);
        else even = t.stride(k) == span;
        span = t.stride(k) * t.size(k);
    }
    // (an expanded axis steps by 0)
    if (!even || inner != D || (rows > 1 && step < D)) return {t.contiguous(), rows, D};
    return {t, rows, rows > 1 ? step : D};
}

// a view whose negation is pending, as the imaginary part of a conjugate, written out: the kernels read memory
Tensor in_memory(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor forward(const Tensor& x, const Tensor& w, const Tensor& b, int64_t D, double eps, Tensor* stats) {
    auto [xr, rows, xs] = rows_of(x, D);
    Tensor y = at::empty(x.sizes(), x.options());
    if (stats) *stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
    const int dt = dtype_of(x), wdt = w.defined() ? dtype_of(w) : b.defined() ? dtype_of(b) : dt;
    const c10::DeviceGuard guard(x.device());
    check_status(pcx.layernorm_forward(dt, wdt, rows, D, xr.const_data_ptr(), xs, address(w), address(b), (float)eps,
                                       y.mutable_data_ptr(), stats ? stats->mutable_data_ptr<float>() : nullptr,
                                       stream_of(x)),
                 "pcx_layernorm_forward");
    return y;
}

// The gradient as a function of x, w and dy: it is not differentiable, and says so when asked to be.
struct LayerNormGradient : torch::autograd::Function<LayerNormGradient> {
    static variable_list forward(AutogradContext*, at::TensorList all, int64_t n) {
        return variable_list(all.begin(), all.begin() + n);
    }
    static variable_list backward(AutogradContext*, const variable_list&) {
        TORCH_CHECK(false, "layer_norm: its gradient is not differentiable");
    }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    // (an absent tensor has no edge: needs_input_grad counts x and those that are there)
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                          const std::optional<Tensor>& bias, int64_t D, double eps) {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        Tensor stats, y = ::forward(x, w, b, D, eps, &stats);
        ctx->saved_data["has_b"] = b.defined();
        ctx->save_for_backward({x, w, stats});
        const Tensor& t = w.defined() ? w : b;
        ctx->saved_data["D"] = D;
        ctx->saved_data["eps"] = eps;
        if (t.defined()) {
            ctx->saved_data["shape"] = t.sizes().vec();
            ctx->saved_data["type"] = (int64_t)t.scalar_type();
        }
        return y;
    }

    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
        const int64_t D = ctx->saved_data["D"].toInt();
        const double eps = ctx->saved_data["eps"].toDouble();
        const bool need_x = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(1);
        const bool need_b = ctx->saved_data["has_b"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1);
        auto [xr, rows, xs] = rows_of(x, D);
        Tensor dx, dw, db, ws;
        if (need_x) dx = at::empty(x.sizes(), x.options());
        const int dt = dtype_of(x);
        int wdt = dt;
        if (need_w || need_b) {
            const auto shape = ctx->saved_data["shape"].toIntVector();
            const auto opt = x.options().dtype((at::ScalarType)ctx->saved_data["type"].toInt());
            if (need_w) dw = at::empty(shape, opt);
            if (need_b) db = at::empty(shape, opt);
            wdt = dtype_of(need_w ? dw : db);
        } else if (w.defined()) {
            wdt = dtype_of(w);
        }
        const c10::DeviceGuard guard(x.device());
        if (rows == 0) {
            if (need_w) dw.zero_();
            if (need_b) db.zero_();
        } else {
            auto [dyr, dyrows, dys] = rows_of(in_memory(grads[0]), D);
            size_t nws = 0;
            if (need_w || need_b) {
                nws = pcx.workspace_bytes(dt, rows, D);
                if (nws) ws = at::empty({(int64_t)nws}, x.options().dtype(at::kByte));
            }
            check_status(pcx.layernorm_backward(dt, wdt, rows, D, xr.const_data_ptr(), xs, address(w), (float)eps,
                                                stats.const_data_ptr<float>(), dyr.const_data_ptr(), dys,
                                                need_x ? dx.mutable_data_ptr() : nullptr,
                                                need_w ? dw.mutable_data_ptr() : nullptr,
                                                need_b ? db.mutable_data_ptr() : nullptr,
                                                nws ? ws.mutable_data_ptr() : nullptr, nws, stream_of(x)),
                         "pcx_layernorm_backward");
        }
        if (at::GradMode::is_enabled()) {  // create_graph
            variable_list all;
            for (const Tensor& t : {dx, dw, db, x, w, grads[0]})
                if (t.defined()) all.push_back(t);
            const int64_t n = dx.defined() + dw.defined() + db.defined();
            const variable_list out = LayerNormGradient::apply(at::TensorList(all), n);
            int64_t k = 0;
            for (Tensor* t : {&dx, &dw, &db})
                if (t->defined()) *t = out[k++];
        }
        return {dx, dw, db, Tensor(), Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, at::IntArrayRef shape, const std::optional<Tensor>& weight,
                  const std::optional<Tensor>& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    TORCH_CHECK(pcx.layernorm_forward, "layer_norm: phoneme_contrast_amd._lib.torch_ops() has not loaded libpcx.so");
    TORCH_CHECK_VALUE(dtype_of(x) >= 0, "layer_norm: float32, bfloat16 or float16 expected, got ", x.scalar_type());
    const int64_t n = (int64_t)shape.size();
    TORCH_CHECK_VALUE(n >= 1 && x.dim() >= n && x.sizes().slice(x.dim() - n) == shape, "layer_norm: input of shape ", x.sizes(),
                      " does not end in ", shape);
    int64_t D = 1;
    for (const int64_t s : shape) D *= s;
    TORCH_CHECK_VALUE(D >= 1 && D <= 32768, "layer_norm: rows of 1 to 32768 values supported, got ", shape);
    for (const Tensor* t : {&w, &b}) {
        if (!t->defined()) continue;
        const char* name = t == &w ? "weight" : "bias";
        TORCH_CHECK_VALUE(t->sizes() == shape, "layer_norm: ", name, " of shape ", t->sizes(), ", ", shape, " expected");
        TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, "layer_norm: ", name,
                          " must be ", x.scalar_type(), " or float32, got ", t->scalar_type());
        TORCH_CHECK(t->device() == x.device(), "layer_norm: ", name, " is on ", t->device(), ", the input on ", x.device(),
                    ": tensors must live on one ROCm GPU");
    }
    TORCH_CHECK_VALUE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                      "layer_norm: weight and bias must have one type");
    TORCH_CHECK_VALUE(eps > 0. && eps < 1e30, "layer_norm: eps must be positive, got ", eps);
    TORCH_CHECK(x.is_cuda(), "layer_norm: tensors must live on a ROCm GPU (got device '", x.device(), "')");
    for (const Tensor* t : {&x, &w, &b})  // (a tensor outside of a forward-mode level has none)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "layer_norm: no forward-mode derivative");
    const Tensor xr = in_memory(x);
    std::optional<Tensor> wc, bc;
    if (w.defined()) wc = in_memory(w).contiguous();
    if (b.defined()) bc = in_memory(b).contiguous();
    if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad())))
        return LayerNorm::apply(xr, wc, bc, D, eps);
    return forward(xr, wc.value_or(Tensor()), bc.value_or(Tensor()), D, eps, nullptr);
}

}  // namespace

// addresses of the entry points, in the order of Entries
extern "C" __attribute__((visibility("default"))) void pcx_torch_bind(void* const* at) {
    pcx.last_error = reinterpret_cast<decltype(pcx.last_error)>(at[0]);
    pcx.workspace_bytes = reinterpret_cast<decltype(pcx.workspace_bytes)>(at[1]);
    pcx.layernorm_forward = reinterpret_cast<decltype(pcx.layernorm_forward)>(at[2]);
    pcx.layernorm_backward = reinterpret_cast<decltype(pcx.layernorm_backward)>(at[3]);
}

TORCH_LIBRARY(pcx, m) {
    m.def("layer_norm(Tensor x, int[] shape, Tensor? weight, Tensor? bias, float eps) -> Tensor");
}
TORCH_LIBRARY_IMPL(pcx, CompositeImplicitAutograd, m) { m.impl("layer_norm", &layer_norm); }
