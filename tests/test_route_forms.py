"""The router's other forms (``moe_route`` with softmax scores, groups, gates as they are or scaled) against 64-bit arithmetic.

Whole numbers are equal: the choice is that of 64 bits, ties to the lower expert.  Gates: fp32 scores (exponential and quotient within
2^-21), their sum and a quotient: 2^-19.  Gradients of the logits: 2^-18 of the sum of their absolute terms, and one rounding to the
logits' type."""
import pytest
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _choose(logits, bias, k, scores, n_groups, top_groups):
    x = logits.detach().double().cpu()
    s = torch.sigmoid(x) if scores == "sigmoid" else torch.softmax(x, -1)
    by = s + (bias.double().cpu() if bias is not None else 0)
    by = torch.where(torch.isnan(by), torch.full_like(by, float("-inf")), by)
    T, E = by.shape
    if n_groups > 1:
        per = by.view(T, n_groups, -1)
        best = per.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        best = torch.where(torch.isnan(best), torch.full_like(best, float("-inf")), best)
        order = best.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        closed = torch.ones(T, n_groups, dtype=torch.bool).scatter_(1, order, False).repeat_interleave(E // n_groups, 1)
    else:
        closed = torch.zeros(T, E, dtype=torch.bool)
    # open experts by falling score, closed ones behind them all (they may be -inf alike)
    order = by.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(1, closed.gather(1, order).int().sort(dim=-1, stable=True).indices)
    return s, order[:, :k]


def _gates(s, top, renormalise, scale):
    g = s.gather(1, top)
    return scale * (g / (g.sum(-1, keepdim=True) + 1e-9) if renormalise else g)


def _check_pairs(r, top, gates, E):
    """Everything that follows from the choice."""
    T, k = top.shape
    flat = top.reshape(-1)
    order = torch.argsort(flat, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k)
    pos, perm = place.view(T, k).sort(dim=1)
    counts = torch.bincount(flat, minlength=E)
    want = dict(top_experts=top.int(), token_indices=order // k, sorted_experts=flat[order], counts=counts, ends=counts.cumsum(0),
                starts=counts.cumsum(0) - counts, pair_pos=pos)
    for name, w in want.items():
        assert r[name].dtype == w.dtype and torch.equal(r[name].cpu(), w), name
    for name, w in (("top_gates", gates), ("sorted_scores", gates.reshape(-1)[order]), ("pair_gate", gates.gather(1, perm))):
        got = r[name].detach().double().cpu()
        assert got.shape == w.shape and ((got - w).abs() <= 2.0 ** -19 * w.abs() + 2.0 ** -149).all(), name


FORMS = [("softmax", 1, 1, True, 1.0), ("softmax", 1, 1, False, 2.5), ("sigmoid", 2, 1, True, 2.5), ("sigmoid", 4, 3, False, 1.0), ("softmax", 4, 2, True, 0.5),
         ("sigmoid", 1, 1, False, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scores,n_groups,top_groups,renormalise,scale", FORMS)
@pytest.mark.parametrize("T,E,k", [(1, 4, 1), (3, 8, 2), (130, 60, 6), (257, 256, 8), (1000, 16, 4), (65, 1024, 32), (33, 384, 5), (4, 12, 3)])
def test_choice_pairs_and_gradient(T, E, k, scores, n_groups, top_groups, renormalise, scale, dtype):
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(T + E)
    logits = (torch.randn(T, E, generator=g) * 1.5).to(dtype).cuda().requires_grad_(True)
    bias = (torch.randn(E, generator=g) * 0.1).cuda() if E % 3 else None
    form = dict(scores=scores, n_groups=n_groups, top_groups=top_groups, renormalise=renormalise, scale=scale)
    r = K.moe_route(logits, bias, k, **form)
    s, top = _choose(logits, bias, k, scores, n_groups, top_groups)
    gates = _gates(s, top, renormalise, scale)
    _check_pairs(r, top, gates, E)
    with torch.no_grad():
        plain = K.moe_route(logits, bias, k, **form)
    for name in r:
        assert torch.equal(plain[name], r[name]), name
    # gradients by slot, in the order of the rows, and by sorted pair
    x = logits.detach().double().cpu().requires_grad_(True)
    s = torch.sigmoid(x) if scores == "sigmoid" else torch.softmax(x, -1)
    mine = _gates(s, top, renormalise, scale)
    perm = top.sort(dim=1).indices
    order = torch.argsort(top.reshape(-1), stable=True)
    d = [torch.randn(T, k, generator=g), torch.randn(T, k, generator=g), torch.randn(T * k, generator=g)]
    for use in ((0,), (1,), (2,), (0, 1, 2)):
        outs = [(r["top_gates"], mine), (r["pair_gate"], mine.gather(1, perm)), (r["sorted_scores"], mine.reshape(-1)[order])]
        got, = torch.autograd.grad([outs[i][0] for i in use], logits, [d[i].cuda() for i in use], retain_graph=True)
        want, = torch.autograd.grad([outs[i][1] for i in use], x, [d[i].double() for i in use], retain_graph=True)
        dg = torch.zeros(T, k, dtype=torch.float64)
        if 0 in use:
            dg += d[0].double().abs()
        if 1 in use:
            dg.scatter_add_(1, perm, d[1].double().abs())
        if 2 in use:
            dg += torch.empty(T * k, dtype=torch.float64).scatter_(0, order, d[2].double().abs()).view(T, k)
        picked = s.detach().gather(1, top)
        dg = dg * abs(scale)
        if renormalise:
            total = picked.sum(-1, keepdim=True) + 1e-9
            dg = (dg + (dg * picked).sum(-1, keepdim=True) / total) / total
        terms = torch.zeros(T, E, dtype=torch.float64).scatter_(1, top, dg)
        if scores == "softmax":
            terms = s.detach() * (terms + (dg * picked).sum(-1, keepdim=True))
        else:
            terms = terms * s.detach()                                 # (1 - s is off by s's rounding, of s)
        tol = 2.0 ** -18 * terms + HALF_STEP[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert got.dtype == dtype
        over = (got.double().cpu() - want).abs() - tol
        assert over.max() <= 0, (use, float(over.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n_groups,top_groups", [(1, 1), (8, 3)])
def test_ties_and_scores_next_to_each_other(scores, n_groups, top_groups):
    """Equal logits, logits a step apart, saturated scores, with and without a bias that undoes the difference."""
    from cinnamon_b200 import kernels as K
    T, E, k = 600, 64, 6
    g = torch.Generator().manual_seed(9)
    base = torch.randint(-2, 3, (T, E), generator=g).float()
    steps = base.clone()
    near = torch.rand(T, E, generator=g)
    steps = torch.where(near < 0.3, torch.nextafter(steps, torch.tensor(10.0)), steps)
    steps = torch.where(near > 0.8, torch.nextafter(steps, torch.tensor(-10.0)), steps)
    for logits in (base, steps, base * 20, torch.zeros(T, E), base.bfloat16()):
        for bias in (torch.zeros(E), torch.randint(0, 2, (E,), generator=g).float() * 2.0 ** -12, None):
            r = K.moe_route(logits.cuda(), bias.cuda() if bias is not None else None, k, scores=scores, n_groups=n_groups, top_groups=top_groups,
                            scale=1.5)
            s, top = _choose(logits, bias, k, scores, n_groups, top_groups)
            assert torch.equal(r["top_experts"].cpu(), top.int())


@pytest.mark.gpu
@pytest.mark.parametrize("n_groups,top_groups", [(1, 1), (4, 2)])
def test_nan_infinities_and_banned_experts(n_groups, top_groups):
    """Biases of -inf ban experts, NaN logits come last; k experts are chosen all the same, none of them twice."""
    from cinnamon_b200 import kernels as K
    T, E, k = 40, 16, 8
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(T, E, generator=g)
    bias = torch.zeros(E)
    bias[torch.tensor([1, 5, 6, 7])] = float("-inf")
    logits[3, 2], logits[4, :] = float("nan"), float("nan")
    logits[5, 8:], logits[6, 3] = float("-inf"), float("inf")
    lowest = torch.finfo(torch.float32).min
    logits[7, :], logits[8, 0:12] = lowest, lowest
    bias2 = torch.full((E,), lowest)
    for b in (bias, bias2):
        r = K.moe_route(logits.cuda(), b.cuda(), k, n_groups=n_groups, top_groups=top_groups, scale=2.0)
        _, top = _choose(logits, b, k, "sigmoid", n_groups, top_groups)
        assert torch.equal(r["top_experts"].cpu(), top.int())
        assert all(len(set(row)) == k for row in r["top_experts"].tolist())
        fine = torch.ones(T, dtype=torch.bool)
        fine[3], fine[4] = False, False
        assert torch.isfinite(r["top_gates"].cpu()[fine]).all()
    r = K.moe_route(logits[9:].cuda(), torch.zeros(E).cuda(), k, scores="softmax", n_groups=n_groups, top_groups=top_groups)
    assert torch.equal(r["top_experts"].cpu(), _choose(logits[9:], torch.zeros(E), k, "softmax", n_groups, top_groups)[1].int())


@pytest.mark.gpu
@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e31])
def test_groups_whose_experts_are_banned(low):
    """Masks of the lowest values: in some groups one expert is left, in some none; biases that cancel in a group's sum."""
    from cinnamon_b200 import kernels as K
    T, E = 300, 64
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(T, E, generator=g)
    bias = torch.randn(E, generator=g) * 0.1
    bias[0:8], bias[9:16], bias[24:31] = low, low, low
    for k, top_groups in ((4, 2), (20, 3), (33 - 1, 4)):
        r = K.moe_route(logits.cuda(), bias.cuda(), k, n_groups=8, top_groups=top_groups, scale=2.0)
        assert torch.equal(r["top_experts"].cpu(), _choose(logits, bias, k, "sigmoid", 8, top_groups)[1].int())
    bias = torch.where(torch.arange(E) % 8 == 0, 4096.0, torch.where(torch.arange(E) % 8 == 1, -4095.0, -5000.0))
    r = K.moe_route(logits.cuda(), bias.cuda(), 4, n_groups=8, top_groups=3, scale=2.0)
    assert torch.equal(r["top_experts"].cpu(), _choose(logits, bias, 4, "sigmoid", 8, 3)[1].int())


@pytest.mark.gpu
@pytest.mark.parametrize("E,n_groups,top_groups,k", [(1, 1, 1, 1), (32, 32, 5, 5), (8, 8, 3, 3), (64, 32, 16, 32), (1024, 32, 1, 32), (96, 3, 1, 32), (512, 4, 1, 32),
                                                     (1024, 8, 8, 32)])
def test_groups_of_one_and_all_of_a_lane(E, n_groups, top_groups, k):
    """Groups of a single expert, every expert of the open groups, and more of the best in one lane than it keeps."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(E)
    for scores in ("sigmoid", "softmax"):
        logits = torch.randn(70, E, generator=g)
        logits[:, :k] += 3.0
        r = K.moe_route(logits.cuda(), None, k, scores=scores, n_groups=n_groups, top_groups=top_groups)
        assert torch.equal(r["top_experts"].cpu(), _choose(logits, None, k, scores, n_groups, top_groups)[1].int())


@pytest.mark.gpu
def test_the_references_form_keeps_its_bits_and_gains_a_gradient():
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(1)
    logits, bias = torch.randn(500, 64, generator=g).cuda(), (torch.randn(64, generator=g) * 0.1).cuda()
    plain = K.moe_route(logits, bias, 4)
    x = logits.clone().requires_grad_(True)
    r = K.moe_route(x, bias, 4)
    for name in plain:
        assert torch.equal(r[name], plain[name]), name
    d = torch.randn(500, 4, device="cuda")
    got, = torch.autograd.grad(r["pair_gate"], x, d)
    y = logits.double().requires_grad_(True)
    s = torch.sigmoid(y).gather(1, plain["top_experts"].long().sort(1).values)
    want, = torch.autograd.grad(s / (s.sum(-1, keepdim=True) + 1e-9), y, d.double())
    assert ((got.double() - want).abs() <= 2.0 ** -17 * d.double().abs().sum(-1, keepdim=True)).all()


@pytest.mark.gpu
def test_no_tokens_strides_streams_and_graphs():
    from cinnamon_b200 import kernels as K
    form = dict(scores="softmax", n_groups=4, top_groups=2, renormalise=False)
    r = K.moe_route(torch.empty(0, 32, device="cuda", requires_grad=True), None, 3, **form)
    assert r["top_experts"].shape == (0, 3) and (r["counts"] == 0).all() and (r["ends"] == 0).all()
    wide = torch.randn(200, 80, device="cuda")
    bias = torch.zeros(32, device="cuda")
    ref = K.moe_route(wide[:, 3:35].contiguous(), bias, 3, **form)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        other = K.moe_route(wide[:, 3:35], bias, 3, **form)
        x = wide[:, 3:35].clone().requires_grad_(True)
        with torch.cuda.graph(graph, stream=side):
            captured = K.moe_route(x, bias, 3, **form)
            grad, = torch.autograd.grad(captured["top_gates"], x, torch.ones(200, 3, device="cuda"))
    torch.cuda.synchronize()
    for name in ref:
        assert torch.equal(other[name], ref[name]), name
    fresh = torch.randn(200, 32, device="cuda")
    with torch.no_grad():
        x.copy_(fresh)
    graph.replay()
    torch.cuda.synchronize()
    y = fresh.clone().requires_grad_(True)
    want = K.moe_route(y, bias, 3, **form)
    for name in ref:
        assert torch.equal(captured[name], want[name]), name
    assert torch.equal(grad, torch.autograd.grad(want["top_gates"], y, torch.ones(200, 3, device="cuda"))[0])


@pytest.mark.gpu
def test_refusals():
    from cinnamon_b200 import kernels as K
    x, b = torch.randn(5, 32, device="cuda"), torch.zeros(32, device="cuda")
    for kw, what in [(dict(scores="tanh"), "scores"), (dict(n_groups=5), "groups"), (dict(n_groups=64), "groups"), (dict(n_groups=4, top_groups=5), "groups"),
                     (dict(n_groups=8, top_groups=1), "out of"), (dict(n_groups=0), "groups")]:
        with pytest.raises(AssertionError, match=what):
            K.moe_route(x, b, 6, **kw)
    for args in ((x, b, 33), (x, b, 0), (x, b[:5], 2), (x[0], b, 2), (x, b.cpu(), 2), (torch.randn(2, 2000, device="cuda"), None, 2)):
        with pytest.raises(AssertionError):
            K.moe_route(*args, scores="softmax")
    a = x.clone().requires_grad_(True)
    with pytest.raises(AssertionError, match="second derivative"):
        torch.autograd.grad(K.moe_route(a, b, 2, scores="softmax")["top_gates"].sum(), a, create_graph=True)


def _block(form, alpha=0.0, d=256, hidden=512):
    from cinnamon_b200 import layers
    torch.manual_seed(3)
    return layers.MoE(16, 1, 4, d, hidden, 2, 0.001, balance_alpha=alpha, router_form=form)


@pytest.mark.gpu
@pytest.mark.parametrize("alpha", [0.0, 0.01])
def test_moe_block_with_a_router_of_groups(alpha):
    """layers.MoE: the native block against the same module taken apart (a hook on the router keeps it from being native)."""
    from cinnamon_b200 import kernels as K, moe
    form = moe.RouterForm(scores="softmax", n_groups=4, top_groups=2, renormalise=False, scale=2.0)
    block = _block(form, alpha).cuda()
    block.expert_bias.copy_(torch.randn(16) * 0.05)
    K.convert_to_fp8(block)
    x = torch.randn(2, 96, 256, device="cuda").bfloat16()
    dy = torch.randn(2, 96, 256, device="cuda")
    results = []
    for hooked in (False, True):
        block.eval()                                                    # (the bias stays as it is)
        hook = block.router.register_forward_hook(lambda *a: None) if hooked else None
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y, balance = block(xi)
        outs = [y] + ([balance] if alpha else [])
        grads = torch.autograd.grad(outs, [xi, block.router.weight, block.routed_experts.w12], [dy] + ([torch.ones_like(balance)] if alpha else []))
        results.append([y.detach(), *grads])
        if hook:
            hook.remove()
    for a, b in zip(*results):
        assert (a.float() - b.float()).norm() <= 2e-2 * b.float().norm()
    assert results[0][2].abs().sum() > 0


@pytest.mark.gpu
def test_serving_layer_with_a_router_of_groups():
    from cinnamon_b200 import moe
    g = torch.Generator().manual_seed(5)
    E, d, I, k, T = 32, 256, 128, 4, 100
    form = moe.RouterForm(n_groups=8, top_groups=3, scale=2.5)
    w12, w3 = (torch.randn(E, 2 * I, d, generator=g) * 0.05).cuda(), (torch.randn(E, d, I, generator=g) * 0.05).cuda()
    router, bias = torch.randn(E, d, generator=g).bfloat16().cuda(), (torch.randn(E, generator=g) * 0.1).cuda()
    layer = moe.ExpertParallelMoE(router, bias, w12, w3, k, router_form=form)
    x = torch.randn(T, d, generator=g).bfloat16().cuda()
    y = layer(x)
    layer.trace = []                                                    # the same layer step by step
    z = layer(x)
    assert torch.equal(y, z)
    r = moe.route(x, router, bias, k, form)
    logits = torch.nn.functional.linear(x, router)
    _, top = _choose(logits, bias, k, "sigmoid", 8, 3)
    assert torch.equal(r.counts.cpu(), torch.bincount(top.reshape(-1), minlength=E))
    plain = moe.ExpertParallelMoE(router, bias, w12, w3, k)(x)
    assert not torch.equal(plain, y)


def test_block_on_the_cpu_and_refusals():
    from cinnamon_b200 import moe
    form = moe.RouterForm(scores="softmax", n_groups=4, top_groups=2, scale=2.0)
    block = _block(form, alpha=0.01, d=32, hidden=64)
    block.eval()
    x = torch.randn(2, 5, 32)
    y, balance = block(x)
    flat = x.view(-1, 32)
    logits = block.router(flat)
    _, top = _choose(logits, block.expert_bias, 4, "softmax", 4, 2)
    s = torch.softmax(logits, -1).gather(1, top)
    gates = 2.0 * s / (s.sum(-1, keepdim=True) + 1e-9)
    want = block.shared_experts[0](flat)
    for e in range(16):
        h1, h2 = torch.nn.functional.linear(flat, block.routed_experts.w12[e]).chunk(2, -1)
        out = torch.nn.functional.linear(torch.nn.functional.silu(h1) * h2, block.routed_experts.w3[e])
        want = want + out * (gates * (top == e)).sum(-1, keepdim=True)
    assert torch.allclose(y.view(-1, 32), want, atol=1e-5, rtol=1e-4) and balance.ndim == 0
    for bad in (dict(n_groups=3), dict(n_groups=8, top_groups=1), dict(scores="max"), dict(n_groups=2, top_groups=3)):
        with pytest.raises(AssertionError):
            _block(moe.RouterForm(**bad))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E", [16, 60, 257])
def test_the_gradient_of_a_single_renormalised_gate_is_what_is_left(E, scores, dtype):
    """The gate is s / (s + 1e-9): its derivative 1e-9 / (s + 1e-9)^2 is far below the rounding of what cancels.  Three quotients and sums in fp32 of
    relative error 2^-23 each, the score's own 2^-21 three times over, 1 - s from a score near 1: 2^-23 / (1 - s)."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(E)
    logits = torch.randn(300, E, generator=g).to(dtype).cuda().requires_grad_(True)
    d = torch.randn(300, 1, generator=g).cuda()
    r = K.moe_route(logits, None, 1, scores=scores, n_groups=1 if scores == "softmax" or E == 257 else 2, scale=2.0)
    got, = torch.autograd.grad(r["top_gates"], logits, d)
    x = logits.detach().double().requires_grad_(True)
    s = (torch.sigmoid(x) if scores == "sigmoid" else torch.softmax(x, -1)).gather(-1, r["top_experts"].long())
    want, = torch.autograd.grad(2.0 * s / (s + 1e-9), x, d.double())
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    tol = want.abs() * (half + 2.0 ** -18 + 2.0 ** -22 / (1 - s.detach()).clamp(min=1e-6)) + 2.0 ** -133
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scores,renormalise", [("softmax", True), ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("gates", ["top_gates", "pair_gate", "sorted_scores"])
def test_outputs_changed_in_place_before_the_backward(gates, scores, renormalise):
    """What the backward reads cannot be changed unnoticed (a sharded caller that makes expert ids local does it); what it does not read can."""
    from cinnamon_b200 import kernels as K
    x = torch.randn(70, 32, device="cuda").requires_grad_(True)
    form = dict(scores=scores, renormalise=renormalise, scale=2.0)
    up = torch.randn(70, 4, device="cuda")

    def call():
        r = K.moe_route(x, None, 4, **form)
        return r, lambda: torch.autograd.grad(r[gates], x, up.view(r[gates].shape))[0]
    want = call()[1]()
    for name in ("top_experts", "sorted_experts", "pair_pos"):
        r, back = call()
        r[name] -= 16
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            back()
    r, back = call()
    for name in ("token_indices", "counts", "starts", "ends"):
        r[name].fill_(-7)
    with torch.no_grad():
        r["top_gates" if gates != "top_gates" else "pair_gate"].zero_()
    assert torch.equal(back(), want)
    # past the versions, ids that there are none of have no part in it
    r, back = call()
    r["top_experts"].data.fill_(1 << 30)
    assert (back() == 0).all()
    for bad in (-1, 70 * 4, 1 << 40):
        r, back = call()
        r["pair_pos"].data.fill_(bad)
        r["sorted_experts"].data.fill_(bad)
        got = back()
        assert torch.equal(got, want) if gates == "top_gates" else (got == 0).all()
    assert K.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,n_groups", [(1, 1), (2, 1), (3, 1), (8, 2), (24, 4), (32, 1), (32, 8)])
@pytest.mark.parametrize("kind", ["banned", "all banned", "underflow", "equal"])
def test_all_experts_are_chosen(kind, E, n_groups, scores):
    """As many as there are: banned experts come last, each once, and so do those whose score is 0 in fp32."""
    from cinnamon_b200 import kernels as K
    T = 300
    g = torch.Generator().manual_seed(E)
    logits = torch.zeros(T, E) if kind == "equal" else torch.randn(T, E, generator=g)
    if kind == "underflow":
        logits[torch.rand(T, E, generator=g) < 0.5] -= 110.0
    for low in (float("-inf"), -1e31, torch.finfo(torch.float32).min):
        bias = torch.full((E,), low if kind == "all banned" else 0.0)
        if kind in ("banned", "equal"):
            bias[::2] = low
        bias = None if kind == "underflow" and low != -1e31 else bias.cuda()
        x = logits.cuda().requires_grad_(True)
        r = K.moe_route(x, bias, E, scores=scores, n_groups=n_groups, top_groups=n_groups, renormalise=False)
        s, top = _choose(logits, bias, E, scores, n_groups, n_groups)
        want = dict(top_experts=top.int(), counts=torch.full((E,), T), sorted_experts=torch.arange(E).repeat_interleave(T),
                    token_indices=torch.arange(T).repeat(E))
        for name, w in want.items():
            assert torch.equal(r[name].cpu(), w), name
        gates = s.gather(1, top)
        assert ((r["top_gates"].detach().double().cpu() - gates).abs() <= 2.0 ** -18 * gates + 2.0 ** -126).all()
        grad, = torch.autograd.grad(r["top_gates"].sum(), x)
        assert torch.isfinite(grad).all()
    assert K.device_status() == 0
