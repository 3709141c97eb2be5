// Output projection + cross entropy (csrc/loss.cu): forward and backward as one native call each, and as a native autograd node.
#include "host.h"

namespace cinnhost {

namespace {

// rows of d elements as the kernels read them: contiguous, 16 bytes apart, on a 16-byte boundary
Tensor rows_of(const Tensor& t) {
    const bool fine = t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
    return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct CrossEntropy { Tensor loss, state, dx_sums, dw_sums; };            // the sums: of the early way, undefined where a gradient is not wanted

// x (T, d), w (V, d) of one 16-bit type, d a multiple of 8; target (T,) int64; reduction 0 none, 1 mean, 2 sum.  early_x, early_w: the gradients whose
// sums are made along the way.
CrossEntropy ce_forward(const Tensor& x, const Tensor& w, const Tensor& target, int64_t ignore, int64_t reduction, bool early_x, bool early_w) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t T = x.size(0), d = x.size(1), V = w.size(0);
    CrossEntropy r;
    r.loss = reduction ? empty({}, at::kFloat, x.device()) : empty({T}, at::kFloat, x.device());
    r.state = empty({api.cinn_linear_ce_state_bytes(T)}, at::kByte, x.device());
    if (early_x) r.dx_sums = empty({api.cinn_linear_ce_early(T, V, d, (int)reduction, 1) / 4}, at::kFloat, x.device());
    if (early_w) r.dw_sums = empty({api.cinn_linear_ce_early(T, V, d, (int)reduction, 2) / 4}, at::kFloat, x.device());
    const int64_t need = api.cinn_linear_ce_workspace_bytes(T, V, d, early_x || early_w ? 1 : 0);
    Tensor ws = empty({need}, at::kByte, x.device());
    check(api.cinn_linear_ce_forward(x.data_ptr(), pitch(x), w.data_ptr(), pitch(w), tag_of(x.scalar_type()), target.data_ptr<int64_t>(), ignore, T, V, d,
                                     (int)reduction, f32(r.loss), r.state.data_ptr(), early_x ? f32(r.dx_sums) : nullptr, early_w ? f32(r.dw_sums) : nullptr,
                                     ws.data_ptr(), need, stream()), "cinn_linear_ce_forward");
    return r;
}

std::tuple<Tensor, Tensor> ce_finish(const Tensor& grad, const Tensor& state, const Tensor& dx_sums, const Tensor& dw_sums, int64_t T, int64_t V, int64_t d,
                                     at::ScalarType type, int64_t reduction) {
    c10::cuda::CUDAGuard guard(state.device());
    const Tensor g = grad.to(at::kFloat).contiguous();
    Tensor dx, dw;
    if (dx_sums.defined()) dx = empty({T, d}, type, state.device());
    if (dw_sums.defined()) dw = empty({V, d}, type, state.device());
    check(api.cinn_linear_ce_finish(tag_of(type), f32(g), T, V, d, (int)reduction, state.data_ptr(), dx.defined() ? f32(dx_sums) : nullptr,
                                    dw.defined() ? f32(dw_sums) : nullptr, dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
                                    stream()), "cinn_linear_ce_finish");
    return {dx, dw};
}

std::tuple<Tensor, Tensor> ce_backward(const Tensor& grad, const Tensor& x, const Tensor& w, const Tensor& state, int64_t reduction, bool want_x, bool want_w) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t T = x.size(0), d = x.size(1), V = w.size(0);
    Tensor g = grad.to(at::kFloat).contiguous(), dx, dw;
    if (want_x) dx = empty({T, d}, x.scalar_type(), x.device());
    if (want_w) dw = empty({V, d}, w.scalar_type(), x.device());
    const int64_t need = api.cinn_linear_ce_workspace_bytes(T, V, d, (want_x ? 1 : 0) | (want_w ? 2 : 0) | 4);
    Tensor ws = empty({need}, at::kByte, x.device());
    check(api.cinn_linear_ce_backward(x.data_ptr(), pitch(x), w.data_ptr(), pitch(w), tag_of(x.scalar_type()), f32(g), T, V, d, (int)reduction,
                                      state.data_ptr(), want_x ? dx.data_ptr() : nullptr, want_w ? dw.data_ptr() : nullptr, ws.data_ptr(), need, stream()),
          "cinn_linear_ce_backward");
    return {dx, dw};
}

struct CrossEntropyNode : public torch::autograd::Function<CrossEntropyNode> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in, const Tensor& target, int64_t ignore,
                          int64_t reduction) {
        const Tensor x = rows_of(x_in), w = rows_of(w_in);
        const bool early = api.cinn_linear_ce_early(x.size(0), w.size(0), x.size(1), (int)reduction, 0);
        const CrossEntropy r = ce_forward(x, w, target, ignore, reduction, early && x_in.requires_grad(), early && w_in.requires_grad());
        if (early) {
            ctx->save_for_backward({r.state, r.dx_sums, r.dw_sums});
            ctx->saved_data["shape"] = std::vector<int64_t>{x.size(0), w.size(0), x.size(1), (int64_t)x.scalar_type()};
        } else {
            ctx->save_for_backward({x, w, r.state});
        }
        ctx->saved_data["early"] = early;
        ctx->saved_data["reduction"] = reduction;
        return r.loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        auto s = ctx->get_saved_variables();
        Tensor dx, dw;
        as_python_error([&] {
            require(!at::GradMode::is_enabled(), "linear_cross_entropy has no second derivative (create_graph=True)");
            check_captured_backward("linear_cross_entropy");
            const int64_t reduction = ctx->saved_data["reduction"].toInt();
            const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
            if (ctx->saved_data["early"].toBool()) {
                const auto n = ctx->saved_data["shape"].toIntVector();
                std::tie(dx, dw) = ce_finish(grads[0], s[0], want_x ? s[1] : Tensor(), want_w ? s[2] : Tensor(), n[0], n[1], n[2], (at::ScalarType)n[3], reduction);
            } else {
                std::tie(dx, dw) = ce_backward(grads[0], s[0], s[1], s[2], reduction, want_x, want_w);
            }
        });
        return {dx, dw, Tensor(), Tensor(), Tensor()};
    }
};

// the operands in the type they are multiplied in, padded to whole 16 bytes; differentiable
std::tuple<Tensor, Tensor, Tensor> ce_operands(const Tensor& x_in, const Tensor& w_in, const Tensor& target_in) {
    require(x_in.is_cuda() && w_in.is_cuda() && target_in.is_cuda(), "Inputs must be on CUDA");
    require(x_in.device() == w_in.device() && x_in.device() == target_in.device(), "linear_cross_entropy: x, weight and target must be on the same device");
    require(x_in.dim() >= 1 && w_in.dim() == 2 && x_in.size(-1) == w_in.size(1), "linear_cross_entropy: x is (..., d) and weight (vocabulary, d)");
    require(w_in.size(0) > 0 && w_in.size(1) > 0, "linear_cross_entropy: weight must not be empty");
    require(target_in.scalar_type() == at::kLong || target_in.scalar_type() == at::kInt, "linear_cross_entropy: targets are int64 or int32");
    require(target_in.sizes() == x_in.sizes().slice(0, x_in.dim() - 1), "linear_cross_entropy: target has one entry for every row of x");
    Tensor x = x_in.reshape({-1, x_in.size(-1)}), w = w_in;
    if (at::autocast::is_autocast_enabled(at::kCUDA)) {
        const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
        x = x.to(type);
        w = w.to(type);
    }
    const auto type = x.scalar_type();
    require(type == w.scalar_type() && (type == at::kBFloat16 || type == at::kHalf),
            "linear_cross_entropy multiplies 16-bit operands: x and weight must both be bfloat16 or both float16 (or autocast must make them so)");
    const int64_t odd = x.size(1) % 8;
    if (odd) {
        x = at::constant_pad_nd(x, {0, 8 - odd});
        w = at::constant_pad_nd(w, {0, 8 - odd});
    }
    return {x, w, target_in.reshape({-1}).to(at::kLong).contiguous()};
}

// The calls below are operators of a compiled graph, which hands over what it is given: everything that the kernels rely on is looked at here.
void check_flat(const Tensor& x, const Tensor& w) {
    require(x.is_cuda() && w.is_cuda(), "Inputs must be on CUDA");
    require(x.device() == w.device(), "linear_cross_entropy: x, weight and target must be on the same device");
    require(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.size(1) > 0 && x.size(1) % 8 == 0 && w.size(0) > 0,
            "linear_cross_entropy: x is (tokens, d) and weight (vocabulary, d), d a multiple of 8");
    require(x.scalar_type() == w.scalar_type() && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf),
            "linear_cross_entropy multiplies 16-bit operands");
}
void check_part(const Tensor& t, const at::Device& dev, at::ScalarType type, int64_t numel) {
    require(t.device() == dev && t.scalar_type() == type && t.numel() == numel && t.is_contiguous(),
            "linear_cross_entropy: not what the forward left for this backward");
}
void check_grad(const Tensor& grad, const at::Device& dev, int64_t numel) {
    require(grad.device() == dev && grad.numel() == numel, "linear_cross_entropy: the loss's gradient does not fit it");
}

}  // namespace

void bind_loss(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("linear_ce_early", [](int64_t T, int64_t V, int64_t d, int64_t reduction, int which) { return api.cinn_linear_ce_early(T, V, d, (int)reduction, which); });
    // (loss, state, sums of dx, sums of dw); what is not made is empty: the sums in the late way, and those of a gradient that is not wanted
    m.def("linear_ce_forward", [](const Tensor& x, const Tensor& w, const Tensor& target, int64_t ignore, int64_t reduction, bool early, bool want_x, bool want_w) {
        check_flat(x, w);
        require(target.device() == x.device(), "linear_cross_entropy: x, weight and target must be on the same device");
        require(target.scalar_type() == at::kLong && target.dim() == 1 && target.size(0) == x.size(0), "linear_cross_entropy: target has one int64 for every row of x");
        CrossEntropy r = ce_forward(rows_of(x), rows_of(w), target.contiguous(), ignore, reduction, early && want_x, early && want_w);
        auto sums = [&](const Tensor& t) { return t.defined() ? t : empty({0}, at::kFloat, x.device()); };
        return std::make_tuple(r.loss, r.state, sums(r.dx_sums), sums(r.dw_sums));
    }, py::arg("x"), py::arg("w"), py::arg("target"), py::arg("ignore"), py::arg("reduction"), py::arg("early"), py::arg("want_x") = true, py::arg("want_w") = true);
    // (dx, dw) of the early and of the late way; one that is not wanted is empty
    auto made = [](const std::tuple<Tensor, Tensor>& r, at::ScalarType type, const at::Device& dev) {
        auto t = [&](const Tensor& g) { return g.defined() ? g : empty({0}, type, dev); };
        return std::make_tuple(t(std::get<0>(r)), t(std::get<1>(r)));
    };
    m.def("linear_ce_finish", [made](const Tensor& grad, const Tensor& state, const Tensor& dx_sums, const Tensor& dw_sums, int64_t T, int64_t V, int64_t d,
                                 at::ScalarType type, int64_t reduction, bool want_x, bool want_w) {
        require(state.is_cuda(), "Inputs must be on CUDA");
        require(T > 0 && V > 0 && d > 0 && d % 8 == 0 && (type == at::kBFloat16 || type == at::kHalf) && (reduction == 1 || reduction == 2),
                "linear_cross_entropy: early gradients are those of a sum or mean over some tokens");
        check_grad(grad, state.device(), 1);
        check_part(state, state.device(), at::kByte, api.cinn_linear_ce_state_bytes(T));
        if (want_x) check_part(dx_sums, state.device(), at::kFloat, api.cinn_linear_ce_early(T, V, d, (int)reduction, 1) / 4);
        if (want_w) check_part(dw_sums, state.device(), at::kFloat, api.cinn_linear_ce_early(T, V, d, (int)reduction, 2) / 4);
        return made(ce_finish(grad, state, want_x ? dx_sums : Tensor(), want_w ? dw_sums : Tensor(), T, V, d, type, reduction), type, state.device());
    });
    m.def("linear_ce_backward", [made](const Tensor& grad, const Tensor& x, const Tensor& w, const Tensor& state, int64_t reduction, bool want_x, bool want_w) {
        check_flat(x, w);
        check_grad(grad, x.device(), reduction ? 1 : x.size(0));
        check_part(state, x.device(), at::kByte, api.cinn_linear_ce_state_bytes(x.size(0)));
        return made(ce_backward(grad, rows_of(x), rows_of(w), state, reduction, want_x, want_w), x.scalar_type(), x.device());
    });
    m.def("linear_cross_entropy", [](const Tensor& x_in, const Tensor& w_in, const Tensor& target_in, int64_t ignore, int64_t reduction) {
        const auto [x, w, target] = ce_operands(x_in, w_in, target_in);
        c10::cuda::CUDAGuard guard(x.device());               // (check_capture asks the current device's stream)
        check_capture("linear_cross_entropy", x_in, w_in);
        const Tensor loss = takes_node(x, w) ? CrossEntropyNode::apply(x, w, target, ignore, reduction)
                                             : ce_forward(rows_of(x), rows_of(w), target, ignore, reduction, false, false).loss;
        return reduction ? loss : loss.view(target_in.sizes());
    });
}

}  // namespace cinnhost
