// Rotary positions of queries and keys (csrc/rotary.cu): one native call, and a native autograd node.
#include "host.h"

namespace cinnhost {

namespace {

struct Form { int64_t start; double magnitude; bool interleaved; };

void check_rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freq) {
    require(q.is_cuda() && positions.is_cuda() && freq.is_cuda() && (!k.defined() || k.is_cuda()), "Inputs must be on CUDA");
    require(q.device() == positions.device() && q.device() == freq.device() && (!k.defined() || k.device() == q.device()),
            "rotary: q, k, positions and inv_freq must be on the same device");
    require(q.dim() == 4 && (!k.defined() || k.dim() == 4), "rotary: q and k are (batch, heads, positions, elements)");
    require(tag_of(q.scalar_type()) >= 0, "rotary: q and k are bfloat16, float16 or float32");
    require(!k.defined() || (k.scalar_type() == q.scalar_type() && k.size(0) == q.size(0) && k.size(2) == q.size(2)),
            "rotary: q and k must agree in type, batch and positions");
    require(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "rotary: positions are int64 or int32");
    const bool flat = positions.dim() == 1, both = positions.dim() == 2;
    require((flat || both) && positions.size(-1) == q.size(2) && (flat || positions.size(0) == q.size(0) || positions.size(0) == 1),
            "rotary: positions are (positions,) or (batch, positions)");
    require(freq.dim() == 1 && freq.numel() >= 1 && (freq.scalar_type() == at::kDouble || freq.scalar_type() == at::kFloat),
            "rotary: inv_freq is one number for every pair, float64 (or float32)");
    require(!(at::GradMode::is_enabled() && freq.requires_grad()), "rotary: inv_freq takes no gradient");
}

Tensor heads_of(const Tensor& t) { return t.stride(-1) == 1 || t.numel() == 0 || t.size(-1) == 1 ? t : t.contiguous(); }

// in[i] -> out[i]; undefined: left out
void run(const Tensor (&in)[2], const Tensor (&out)[2], const Tensor& positions, const Tensor& freq, const Form& f, bool inverse) {
    const void* from[2] = {};
    void* to[2] = {};
    int64_t strides[2][6] = {}, heads[2] = {}, d[2] = {}, start[2] = {};
    const Tensor* any = nullptr;
    for (int i = 0; i < 2; ++i) {
        if (!in[i].defined() || in[i].numel() == 0) continue;
        any = &in[i];
        from[i] = in[i].data_ptr();
        to[i] = out[i].data_ptr();
        for (int s = 0; s < 3; ++s) { strides[0][3 * i + s] = in[i].stride(s); strides[1][3 * i + s] = out[i].stride(s); }
        heads[i] = in[i].size(1);
        d[i] = in[i].size(3);
        start[i] = f.start < 0 ? d[i] + f.start : f.start;
    }
    if (!any) return;
    const bool by_batch = positions.dim() == 2 && positions.size(0) > 1;
    check(api.cinn_rotary(from, to, strides[0], strides[1], heads, d, start, tag_of(any->scalar_type()), any->size(0), any->size(2),
                          positions.data_ptr<int64_t>(), by_batch ? positions.stride(0) : 0, positions.stride(-1), freq.data_ptr<double>(), freq.numel(),
                          f.interleaved, inverse, (float)f.magnitude, stream()), "cinn_rotary");
}

std::array<Tensor, 2> turned(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& freq, const Form& f, bool inverse) {
    const Tensor in[2] = {q.defined() ? heads_of(q) : q, k.defined() ? heads_of(k) : k};
    const Tensor out[2] = {q.defined() ? at::empty_like(in[0]) : q, k.defined() ? at::empty_like(in[1]) : k};
    run(in, out, positions, freq, f, inverse);
    return {out[0], out[1]};
}

struct RotaryNode : public torch::autograd::Function<RotaryNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const c10::optional<Tensor>& k_in,
                                                  const Tensor& positions, const Tensor& freq, const Form* f) {
        const Tensor k = k_in.has_value() ? *k_in : Tensor();
        c10::cuda::CUDAGuard guard(positions.device());
        ctx->save_for_backward({positions, freq});
        ctx->saved_data["start"] = f->start;
        ctx->saved_data["magnitude"] = f->magnitude;
        ctx->saved_data["interleaved"] = f->interleaved;
        ctx->set_materialize_grads(false);
        const auto r = turned(q, k, positions, freq, *f, false);
        if (k.defined()) return {r[0], r[1]};
        return {r[0]};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        auto s = ctx->get_saved_variables();
        std::array<Tensor, 2> r;
        as_python_error([&] {
            require(!at::GradMode::is_enabled(), "rotary has no second derivative (create_graph=True)");
            c10::cuda::CUDAGuard guard(s[0].device());
            check_captured_backward("rotary");
            const Form f{ctx->saved_data["start"].toInt(), ctx->saved_data["magnitude"].toDouble(), ctx->saved_data["interleaved"].toBool()};
            r = turned(ctx->needs_input_grad(0) ? grads[0] : Tensor(), grads.size() > 1 && ctx->needs_input_grad(1) ? grads[1] : Tensor(), s[0], s[1], f, true);
        });
        return {r[0], r[1], Tensor(), Tensor(), Tensor()};
    }
};

}  // namespace

void bind_rotary(pybind11::module_& m) {
    using OptT = c10::optional<Tensor>;
    using Pair = std::tuple<Tensor, OptT>;
    m.def("rotary", [](const Tensor& q, const OptT& k_in, const Tensor& positions_in, const Tensor& freq_in, bool interleaved, int64_t start,
                       double magnitude, bool inverse) -> Pair {
        const Tensor k = k_in.has_value() ? *k_in : Tensor();
        check_rotary(q, k, positions_in, freq_in);
        c10::cuda::CUDAGuard guard(q.device());
        const Tensor positions = positions_in.to(at::kLong), freq = freq_in.detach().to(at::kDouble).contiguous();
        const Form f{start, magnitude, interleaved};
        std::array<Tensor, 2> r;
        check_capture("rotary", q, k);
        if (!inverse && (k.defined() ? takes_node(q, k) : takes_node(q))) {
            const auto v = RotaryNode::apply(q, k.defined() ? c10::optional<Tensor>(k) : c10::nullopt, positions, freq, &f);
            r = {v[0], v.size() > 1 ? v[1] : Tensor()};
        } else {
            r = turned(q, k, positions, freq, f, inverse);
        }
        return {r[0], r[1].defined() ? OptT(r[1]) : OptT()};
    });
    m.def("rotary_", [](const Tensor& q, const OptT& k_in, const Tensor& positions_in, const Tensor& freq_in, bool interleaved, int64_t start, double magnitude) {
        const Tensor k = k_in.has_value() ? *k_in : Tensor();
        check_rotary(q, k, positions_in, freq_in);
        c10::cuda::CUDAGuard guard(q.device());
        const Tensor both[2] = {q, k};
        for (const Tensor& t : both) {
            if (!t.defined()) continue;
            require(!(at::GradMode::is_enabled() && t.requires_grad()), "rotary_ is not differentiable: use rotary, or torch.no_grad()");
            require(!t.is_inference() || !at::GradMode::is_enabled(), "rotary_: an inference tensor cannot be changed in place outside of inference mode");
            require(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, "rotary_: the elements of a head must be contiguous");
            for (int64_t i = 0; i < 3; ++i) require(t.size(i) <= 1 || t.stride(i) != 0, "rotary_: an expanded tensor cannot be rotated in place");
        }
        require(!k.defined() || q.numel() == 0 || k.numel() == 0 || q.data_ptr() != k.data_ptr(), "rotary_: q and k must not be the same memory");
        run(both, both, positions_in.to(at::kLong), freq_in.detach().to(at::kDouble).contiguous(), Form{start, magnitude, interleaved}, false);
        for (const Tensor& t : both)
            if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    });
}

}  // namespace cinnhost
