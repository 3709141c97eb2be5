// The MoE layer on one GPU, forward only (moe.ExpertParallelMoE): router, routing, routed experts, shared expert and the
// combine pass as one native call.  Generating for 64 sequences the layer is 0.7 ms of kernels; driven from Python, its
// calls took 0.47 ms of host time, more than the kernels around the grouped GEMMs could hide.
#include "host.h"

namespace cinnhost {

Quantised rowwise(const Tensor& x, bool round_scale, int div) {
    const int64_t M = x.size(0), K = x.size(1);
    Quantised r{empty({M, K}, F8, x.device()), empty({M, up(K, 128)}, at::kFloat, x.device())};
    check(api.cinn_quant_rowwise(x.data_ptr(), tag_of(x.scalar_type()), M, K, x.stride(0), x.stride(1), r.q.data_ptr(), f32(r.s), 128,
                                 round_scale, div, stream()), "cinn_quant_rowwise");
    return r;
}

Quantised swiglu_quantised(const Tensor& h12, int div) {
    const int64_t T = h12.size(0), I = h12.size(1) / 2;
    Quantised r{empty({T, I}, F8, h12.device()), empty({T, up(I, 128)}, at::kFloat, h12.device())};
    check(api.cinn_swiglu_quant_rowwise(h12.data_ptr(), tag_of(h12.scalar_type()), T, I, r.q.data_ptr(), f32(r.s), div, stream()),
          "cinn_swiglu_quant_rowwise");
    return r;
}

Tensor grouped(const Quantised& x, const Quantised& w, const Tensor& starts, const Tensor& ends, at::ScalarType type) {
    const int64_t T = x.q.size(0), E = w.q.size(0), d_out = w.q.size(1), d_in = w.q.size(2);
    Tensor out = empty({T, d_out}, type, x.q.device());
    check(api.cinn_fp8_grouped_gemm(x.q.data_ptr(), f32(x.s), w.q.data_ptr(), f32(w.s), starts.data_ptr<int64_t>(),
                                    ends.data_ptr<int64_t>(), E, T, d_in, d_out, out.data_ptr(), tag_of(type), stream()),
          "cinn_fp8_grouped_gemm");
    return out;
}

void check_layer(const Tensor& x, const Tensor& router, const Tensor& bias, const Quantised& w12, const Quantised& w3) {
    const auto dev = x.device();
    require(x.is_cuda() && router.is_cuda() && bias.is_cuda(), "Inputs must be on CUDA");
    require(router.device() == dev && bias.device() == dev && w12.q.device() == dev && w3.q.device() == dev && w12.s.device() == dev &&
                w3.s.device() == dev, "MoE: input, router and experts must be on the same device");
    const int64_t E = router.size(0), d = x.size(1);
    require(router.size(1) == d && bias.numel() == E && w12.q.size(0) == E && w3.q.size(0) == E && w12.q.size(2) == d &&
                w3.q.size(1) == d && w12.q.size(1) == 2 * w3.q.size(2), "MoE: the widths of input, router and experts do not fit together");
}

Routes route(const Tensor& logits_in, const Tensor& bias, int64_t top_k, const RouteForm& form, Tensor* gates_by_slot) {
    const Tensor logits = readable(logits_in).contiguous(), b = bias.defined() ? bias.to(at::kFloat).contiguous() : bias;
    const int64_t T = logits.size(0), E = logits.size(1);
    const at::Device dev = logits.device();
    Routes r;
    r.pairs = T * top_k;
    r.E = E;
    r.longs = empty({3 * r.pairs + 3 * E}, at::kLong, dev);
    r.floats = empty({2 * r.pairs}, at::kFloat, dev);
    r.top = empty({r.pairs}, at::kInt, dev);
    const int64_t need = form.reference ? api.cinn_moe_route_workspace_ints(T, (int)E) : api.cinn_moe_route_form_workspace_ints(T, (int)E);
    Tensor ws = empty({std::max<int64_t>(1, need)}, at::kInt, dev);
    Tensor top_gates = empty({r.pairs}, at::kFloat, dev);
    if (gates_by_slot) *gates_by_slot = top_gates;
    if (form.reference)
        check(api.cinn_moe_route_ranges(logits.data_ptr(), tag_of(logits.scalar_type()), f32(b), T, (int)E, (int)top_k, ws.data_ptr<int>(),
                                        r.top.data_ptr<int>(), f32(top_gates), r.token_indices(), f32(r.floats), r.sorted_experts(),
                                        r.part(3 * r.pairs), r.part(3 * r.pairs + E), r.part(3 * r.pairs + 2 * E), r.pos(), r.gates(),
                                        stream()), "cinn_moe_route");
    else
        check(api.cinn_moe_route_form(logits.data_ptr(), tag_of(logits.scalar_type()), b.defined() ? f32(b) : nullptr, T, (int)E, (int)top_k,
                                      (int)form.scores, (int)form.n_groups, (int)form.top_groups, form.renormalise, (float)form.scale, ws.data_ptr<int>(),
                                      r.top.data_ptr<int>(), f32(top_gates), r.token_indices(), f32(r.floats), r.sorted_experts(),
                                      r.part(3 * r.pairs), r.part(3 * r.pairs + E), r.part(3 * r.pairs + 2 * E), r.pos(), r.gates(),
                                      stream()), "cinn_moe_route");
    return r;
}

// quantised tokens to the rows of their pairs
Quantised spread(const Quantised& x, const Routes& r, int64_t top_k) {
    const int64_t T = x.q.size(0), d = x.q.size(1), ns = x.s.size(1);
    Quantised rows{empty({r.pairs, d}, F8, x.q.device()), empty({r.pairs, ns}, at::kFloat, x.q.device())};
    check(api.cinn_spread_rows(x.q.data_ptr(), f32(x.s), r.pos(), rows.q.data_ptr(), f32(rows.s), T, r.pairs, (int)top_k, d, ns, stream()),
          "cinn_spread_rows");
    return rows;
}

namespace {

// A GEMM that is not cut along K: a rank of an expert-parallel job runs the shared expert on its share of the tokens, and a token
// gets the same bits there as on one GPU with all of them.  (Cut along K, the layer takes 910 us instead of 916 for 64 tokens of
// 7168 and 256 experts.)
Tensor gemm_whole(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, int64_t M, int64_t N, int64_t K) {
    Tensor out = empty({M, N}, at::kBFloat16, a.device());
    check(api.cinn_fp8_gemm_ws(a.data_ptr(), f32(sa), sa.stride(0), b.data_ptr(), f32(sb), sb.stride(1), sb.stride(0), out.data_ptr(), M, N, K, 0,
                               TAG_BF16, nullptr, 0, stream()), "cinn_fp8_gemm");
    return out;
}

// x (T, d), contiguous; router (E, d) in the type the logits are computed in; the weights as FP8Experts and FP8SwiGLU hold
// them.  Returns (T, d) fp32.
Tensor forward(const Tensor& x, const Tensor& router, const Tensor& bias, int64_t top_k, const Quantised& w12, const Quantised& w3,
               const Quantised& sw12, const Quantised& sw3, bool shared_round, int div, const RouteForm& form) {
    check_layer(x, router, bias, w12, w3);
    require(!sw12.q.defined() || (sw12.q.device() == x.device() && sw12.q.size(1) == x.size(1) && sw3.q.size(0) == x.size(1) &&
                                  sw12.q.size(0) == 2 * sw3.q.size(1)), "MoE: the shared expert does not fit the input");
    c10::cuda::CUDAGuard guard(x.device());
    at::NoGradGuard no_grad;
    const at::Device dev = x.device();
    const int64_t T = x.size(0), d = x.size(1), E = router.size(0);
    const Quantised xq = rowwise(x, false, div);
    Tensor shared;
    if (sw12.q.defined()) {
        const Quantised xs = shared_round ? rowwise(x, true, div) : xq;
        const int64_t I2 = sw12.q.size(0);
        const Quantised h = swiglu_quantised(gemm_whole(xs.q, xs.s, sw12.q, sw12.s, T, I2, d), div);
        shared = gemm_whole(h.q, h.s, sw3.q, sw3.s, T, d, I2 / 2);
    }
    Tensor logits = at::mm(x, router.to(x.scalar_type()).t());
    const Routes r = route(logits, bias, top_k, form);
    const Tensor starts = r.starts(), ends = r.ends();
    const int64_t pairs = r.pairs, *pos = r.pos();
    Quantised rows = spread(xq, r, top_k);
    Tensor h12 = grouped(rows, w12, starts, ends);
    rows = Quantised{};
    const Quantised h = swiglu_quantised(h12, div);
    h12.reset();
    const Tensor out = grouped(h, w3, starts, ends);
    Tensor y = empty({T, d}, at::kFloat, dev);
    if (shared.defined())
        check(api.cinn_moe_combine_add(out.data_ptr(), TAG_BF16, pos, r.gates(), shared.data_ptr(), TAG_BF16, f32(y), T, pairs,
                                       (int)top_k, d, stream()), "cinn_moe_combine_add");
    else
        check(api.cinn_moe_combine(out.data_ptr(), TAG_BF16, pos, r.gates(), f32(y), T, pairs, (int)top_k, d, stream()),
              "cinn_moe_combine");
    return y;
}

}  // namespace

namespace {

struct RouteCall {
    Tensor bias;
    int64_t top_k;
    RouteForm form;
    Routes out;
    Tensor experts, sorted_experts, pos;                     // as the caller gets them
    void parts(int64_t T) {
        experts = part_of(out.top, 0, {T, top_k});
        sorted_experts = part_of(out.longs, out.pairs, {out.pairs});
        pos = part_of(out.longs, 2 * out.pairs, {T, top_k});
    }
};

// gates by slot, in the order of pair_pos and by sorted pair, from the logits
struct RouteNode : public torch::autograd::Function<RouteNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits_in, RouteCall* c) {
        c10::cuda::CUDAGuard guard(logits_in.device());
        at::AutoDispatchBelowAutograd below;
        const Tensor logits = readable(logits_in).contiguous();
        Tensor top;
        c->out = route(logits, c->bias, c->top_k, c->form, &top);
        const Routes& r = c->out;
        const int64_t T = logits.size(0);
        // the caller's own tensors: what they are changed to in place is not what was chosen, and their versions tell
        c->parts(T);
        ctx->save_for_backward({logits, c->experts, c->sorted_experts, c->pos});
        ctx->saved_data["n"] = std::vector<int64_t>{c->top_k, c->form.scores, c->form.renormalise, (int64_t)logits_in.scalar_type()};
        ctx->saved_data["scale"] = c->form.scale;
        ctx->set_materialize_grads(false);
        return {part_of(top, 0, {T, c->top_k}), part_of(r.floats, r.pairs, {T, c->top_k}), part_of(r.floats, 0, {r.pairs})};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const auto n = ctx->saved_data["n"].toIntVector();
        Tensor d;
        as_python_error([&] {
            require(!at::GradMode::is_enabled(), "moe_route has no second derivative (create_graph=True)");
            const Tensor& logits = s[0];
            c10::cuda::CUDAGuard guard(logits.device());
            check_captured_backward("moe_route");
            const int64_t T = logits.size(0), E = logits.size(1);
            Tensor g[3];
            for (int i = 0; i < 3; ++i)
                if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).contiguous();
            auto at = [&](int i) { return g[i].defined() ? f32(g[i]) : nullptr; };
            d = empty({T, E}, logits.scalar_type(), logits.device());
            check(api.cinn_moe_route_form_backward(logits.data_ptr(), tag_of(logits.scalar_type()), s[1].data_ptr<int>(), s[2].data_ptr<int64_t>(),
                                                   s[3].data_ptr<int64_t>(), at(0), at(1), at(2), T, (int)E, (int)n[0], (int)n[1], (int)n[2], (float)ctx->saved_data["scale"].toDouble(), d.data_ptr(),
                                                   stream()), "cinn_moe_route backward");
            d = d.to((at::ScalarType)n[3]);
        });
        return {d, Tensor()};
    }
};

}  // namespace

void bind_moe(pybind11::module_& m) {
    using OptT = c10::optional<Tensor>;
    m.def("moe_route", [](const Tensor& logits, const OptT& bias, int64_t top_k, const RouteOptions& form) {
        require(logits.is_cuda() && (!bias.has_value() || bias->is_cuda()), "Inputs must be on CUDA");
        require(logits.dim() == 2, "logits must be (tokens, experts)");
        require(!bias.has_value() || (bias->device() == logits.device() && bias->dim() == 1 && bias->size(0) == logits.size(1)),
                "moe_route: bias is one number for every expert, on the logits' device");
        require(top_k >= 1 && top_k <= 32, "moe_route: 1 to 32 experts of a token");
        c10::cuda::CUDAGuard guard(logits.device());
        RouteCall c{bias.has_value() ? bias->detach() : Tensor(), top_k, route_form(form), {}};
        const int64_t T = logits.size(0), E = logits.size(1), pairs = T * top_k;
        Tensor top, pair, sorted;
        check_capture("moe_route", logits);
        if (takes_node(logits)) {
            const auto v = RouteNode::apply(logits, &c);
            top = v[0]; pair = v[1]; sorted = v[2];
        } else {
            c.out = route(logits, c.bias, top_k, c.form, &top);
            c.parts(T);
            top = part_of(top, 0, {T, top_k});
            pair = part_of(c.out.floats, pairs, {T, top_k});
            sorted = part_of(c.out.floats, 0, {pairs});
        }
        const Routes& r = c.out;
        pybind11::dict out;
        out["top_experts"] = c.experts;
        out["top_gates"] = top;
        out["token_indices"] = part_of(r.longs, 0, {pairs});
        out["sorted_scores"] = sorted;
        out["sorted_experts"] = c.sorted_experts;
        out["counts"] = r.counts();
        out["starts"] = r.starts();
        out["ends"] = r.ends();
        out["pair_pos"] = c.pos;
        out["pair_gate"] = pair;
        return out;
    });
    m.def("moe_forward", [](const Tensor& x, const Tensor& router, const Tensor& bias, int64_t top_k, const Tensor& w12_q, const Tensor& w12_s,
                            const Tensor& w3_q, const Tensor& w3_s, const OptT& sw12_q, const OptT& sw12_s, const OptT& sw3_q,
                            const OptT& sw3_s, bool shared_round, int div, const RouteOptions& form) {
        auto get = [](const OptT& t) { return t.has_value() ? *t : Tensor(); };
        return forward(x, router, bias, top_k, {w12_q, w12_s}, {w3_q, w3_s}, {get(sw12_q), get(sw12_s)}, {get(sw3_q), get(sw3_s)},
                       shared_round, div, route_form(form));
    });
}

}  // namespace cinnhost
