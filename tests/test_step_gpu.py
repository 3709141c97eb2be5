"""The operators around the framework's layers, together as a training step uses them: rotary positions in front of sparse attention, a
router of groups in the MoE block, and the head's cross entropy; and the same under torch.compile.

The step through autograd against the step taken apart, every operator called by itself with the gradient that comes back to it: the same bits,
except behind sparse attention's keys and values, whose gradients are sums in no fixed order."""
import gc
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


class Step(nn.Module):
    def __init__(self, d=256, heads=4, d_head=96, rot=32, vocab=1000):
        super().__init__()
        from cinnamon_b200 import kernels as K, layers, moe
        self.K, self.heads, self.rot = K, heads, rot
        self.q = nn.Linear(d, heads * d_head, bias=False)
        self.k = nn.Linear(d, heads * d_head, bias=False)
        self.v = nn.Linear(d, heads * 64, bias=False)
        self.o = nn.Linear(heads * 64, d, bias=False)
        form = moe.RouterForm(scores="softmax", n_groups=4, top_groups=2, scale=2.0)
        self.moe = layers.MoE(16, 1, 4, d, 512, 2, 0.001, router_form=form)
        K.convert_to_fp8(self.moe)
        self.head = nn.Linear(d, vocab, bias=False)
        freq, self.magnitude = K.rotary_frequencies(rot, scaling="yarn", factor=4.0, original_len=512)
        self.register_buffer("inv_freq", freq)

    def split(self, t):
        return t.unflatten(-1, (self.heads, -1)).transpose(1, 2)

    def project(self, x):
        return self.split(self.q(x)), self.split(self.k(x)), self.split(self.v(x))

    def rotate(self, q, k, positions):
        return self.K.rotary(q, k, positions, self.inv_freq, start=-self.rot, magnitude=self.magnitude)

    def attend(self, q, k, v, idx):
        return self.K.sparse_attention(q, k, v, idx)[0].transpose(1, 2).flatten(2)

    def mix(self, x, a):
        h = x + self.o(a)
        return h + self.moe(h)[0]

    def loss(self, h, target):
        return self.K.linear_cross_entropy(h, self.head.weight, target)

    def forward(self, x, positions, idx, target):
        q, k, v = self.project(x)
        q, k = self.rotate(q, k, positions)
        return self.loss(self.mix(x, self.attend(q, k, v, idx)), target)


def _data(d=256, vocab=1000, B=2, L=100, picks=24):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(B, L, d, generator=g).cuda()
    idx = (torch.rand(B, L, picks, generator=g) * (torch.arange(L).view(1, L, 1) + 1)).long().cuda()
    target = torch.randint(0, vocab, (B, L), generator=g)
    target[0, :30], target[1, -9:] = -100, -100                        # a prompt, and padding
    positions = torch.arange(L) + torch.tensor([[0], [70000]])
    return x, positions.cuda(), idx, target.cuda()


def _close(a, b, what):
    assert (a.float() - b.float()).norm() <= 2e-2 * b.float().norm(), what


def test_step_is_its_operators():
    torch.manual_seed(1)
    step = Step().cuda().eval()
    x, positions, idx, target = _data()
    x.requires_grad_(True)
    params = dict(step.named_parameters())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = step(x, positions, idx, target)
    grads = dict(zip(["x", *params], torch.autograd.grad(loss, [x, *params.values()])))

    leaf = lambda t: t.detach().requires_grad_(True)                    # noqa: E731
    with torch.autocast("cuda", dtype=torch.bfloat16):
        parts = [leaf(t) for t in step.project(x)]
        turned = step.rotate(parts[0], parts[1], positions)
        q, k, v = leaf(turned[0]), leaf(turned[1]), parts[2]
        a = step.attend(q, k, v, idx)
        la = leaf(a)
        h = step.mix(x, la)
        lh = leaf(h)
        again = step.loss(lh, target)
    assert torch.equal(again, loss)
    gh, g_head = torch.autograd.grad(again, [lh, params["head.weight"]])
    assert torch.equal(g_head, grads["head.weight"])
    assert (gh[0, :30] == 0).all() and (gh[1, -9:] == 0).all() and (gh[0, 30:] != 0).any(-1).all()
    inner = [n for n in params if n.startswith(("moe.", "o."))]
    back = torch.autograd.grad(h, [la, *(params[n] for n in inner)], gh)
    for n, g in zip(inner, back[1:]):
        assert torch.equal(g, grads[n]), n
    gq, gk, gv = torch.autograd.grad(a, [q, k, v], back[0])
    dq, dk = torch.autograd.grad(turned, parts[:2], [gq, gk])
    with torch.autocast("cuda", dtype=torch.bfloat16):
        projected = step.project(x)
    weights = torch.autograd.grad(projected, [params["q.weight"], params["k.weight"], params["v.weight"]], [dq, dk, gv])
    for n, g in zip(("q.weight", "k.weight", "v.weight"), weights):
        _close(g, grads[n], n)
    assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in grads.values())
    assert step.K.device_status() == 0


def test_step_captured_and_replayed():
    torch.manual_seed(2)
    step = Step().cuda().eval()
    x, positions, idx, target = _data()
    params = list(step.parameters())

    def run():
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            loss = step(x, positions, idx, target)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
    torch.cuda.current_stream().wait_stream(side)
    x2, _, _, target2 = _data()
    with torch.no_grad():
        x.copy_(x2.flip(0)), target.copy_(target2.flip(0)), positions.copy_(positions.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    want = run()
    assert torch.equal(out[0], want[0])
    for a, b, (name, _) in zip(out[1:], want[1:], step.named_parameters()):
        _close(a, b, name)


@pytest.mark.parametrize("op", ["loss", "loss_padded", "rotary", "route", "route_reference"])
def test_capture_beside_a_living_graph_of_the_default_stream_is_refused(op):
    """Its backward pass would wait for the default stream, which no capture may."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(4)
    d = 70 if op == "loss_padded" else 64
    x, w = (torch.randn(40, d, generator=g).cuda().bfloat16().requires_grad_(True) for _ in range(2))
    q = torch.randn(1, 2, 40, 64, generator=g).cuda().requires_grad_(True)
    target, positions, bias = torch.arange(40, device="cuda"), torch.arange(40, device="cuda"), torch.zeros(d, device="cuda")
    freq, _ = K.rotary_frequencies(32, device="cuda")
    calls = {"loss": lambda: K.linear_cross_entropy(x, w, target), "loss_padded": lambda: K.linear_cross_entropy(x, w, target),
             "rotary": lambda: K.rotary(q, q.detach(), positions, freq)[0].sum(),
             "route": lambda: K.moe_route(x, bias, 2, scores="softmax")["top_gates"].sum(),
             "route_reference": lambda: K.moe_route(x, bias, 2)["top_gates"].sum()}
    leaves = [q] if op == "rotary" else [x] if op.startswith("route") else [x, w]
    call = calls[op]
    earlier = call()
    want = torch.autograd.grad(earlier, leaves, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with pytest.raises(AssertionError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                call()
        with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):    # (without gradients there is nothing to refuse)
            call()
        del earlier
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(call(), leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert K.device_status() == 0


@pytest.mark.parametrize("L,d", [(40, 100), (1200, 1025)])               # (the second: gradients made early)
def test_cross_entropy_and_rotary_compile_as_one_graph(L, d):
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(2, L, d, generator=g).cuda(), (torch.randn(300, d, generator=g) * 0.1).cuda()
    target = torch.randint(0, 300, (2, L), generator=g).cuda()
    target[0, :7] = -100
    q, k = (torch.randn(2, h, L, 64, generator=g).bfloat16().cuda() for h in (4, 1))
    freq, _ = K.rotary_frequencies(32, device="cuda")
    positions = torch.arange(L, device="cuda") + 1000

    def head(x, w):
        return K.linear_cross_entropy(x, w, target), K.linear_cross_entropy(x, w, target, reduction="none")

    def turn(q, k):
        return K.rotary(q, k, positions, freq, interleaved=True, start=16, magnitude=1.5)

    results = []
    for compiled in (False, True):
        torch._dynamo.reset()
        f, r = (torch.compile(head, fullgraph=True), torch.compile(turn, fullgraph=True)) if compiled else (head, turn)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, q, k)]
        with torch.autocast("cuda", dtype=torch.bfloat16):
            mean, each = f(*leaves[:2])
        oq, ok = r(*leaves[2:])
        grads = torch.autograd.grad([mean, each, oq, ok], leaves, [torch.ones_like(mean), each.detach(), q, k])
        results.append([mean.detach(), each.detach(), oq.detach(), ok.detach(), *grads])
    for a, b in zip(*results):
        assert a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("dynamic", [True, None])
def test_compiled_loss_over_many_token_counts(dynamic):
    """One function traced for any number of tokens, through the border of the gradients that are made in the forward (at a width they are made
    for), against 64 bits; with and without a frozen weight, and the tokens' losses to the bit."""
    from cinnamon_b200 import kernels as K
    from test_loss_gpu import _inputs, _oracle, _within

    def mean(x, w, t):
        return K.linear_cross_entropy(x, w, t)

    def each(x, w, t):
        return K.linear_cross_entropy(x, w, t, reduction="none")

    torch._dynamo.reset()
    f, e = torch.compile(mean, fullgraph=True, dynamic=dynamic), torch.compile(each, fullgraph=True, dynamic=dynamic)
    for T in (130, 257, 2300, 150, 1, 2049):
        x, w, target = _inputs(T, 300, 1024, torch.bfloat16, seed=T)
        x.requires_grad_(True)
        assert torch.equal(e(x.detach(), w, target), each(x.detach(), w, target))
        want = _oracle(x.detach(), w, target, torch.full((T,), 1 / T, device="cuda"), early=T >= 2048)
        for frozen in (False, True):
            w = w.detach().requires_grad_(not frozen)
            loss = f(x, w, target)
            grads = torch.autograd.grad(loss, [x] if frozen else [x, w])
            _within(loss.detach(), want[0].sum() / T, want[1].sum() / T + 2.0 ** -23 * want[0].sum() / T, "loss")
            _within(grads[0], want[2], want[3], "grad_x")
            if not frozen:
                _within(grads[1], want[4], want[5], "grad_w")
    assert K.device_status() == 0


def test_compiled_refusals():
    """What the eager call refuses is refused under torch.compile too."""
    from cinnamon_b200 import kernels as K
    x, w = torch.zeros(5, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(7, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(5, device="cuda", dtype=torch.int64)
    f = torch.compile(lambda x, w, t: K.linear_cross_entropy(x, w, t))
    for args in ((x, w, t.float()), (x, w, t[:4]), (x.float(), w, t), (x, w[:, :56], t)):
        torch._dynamo.reset()
        with pytest.raises(Exception, match="linear_cross_entropy"):
            f(*args)
    assert torch.isfinite(f(x, w, t.int()))


def test_compiled_rotary_refuses_a_gradient_of_the_frequencies():
    from cinnamon_b200 import kernels as K
    q, p = torch.zeros(1, 2, 5, 64, device="cuda"), torch.arange(5, device="cuda")
    freq = K.rotary_frequencies(32, device="cuda")[0].requires_grad_(True)
    torch._dynamo.reset()
    f = torch.compile(lambda q, freq: K.rotary(q, None, p, freq)[0])
    with pytest.raises(Exception, match="takes no gradient"):
        f(q, freq)
    with torch.no_grad():
        assert torch.equal(f(q, freq), q)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_compiled_loss_of_targets_with_strides(dtype):
    """A column, every other token, one target for all: read as the eager call reads them."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(6)
    x, w = torch.randn(90, 64, generator=g).cuda().bfloat16(), torch.randn(300, 64, generator=g).cuda().bfloat16()
    table = torch.randint(0, 300, (180, 3), generator=g).cuda().to(dtype)
    call = lambda x, w, t: K.linear_cross_entropy(x, w, t, reduction="none")      # noqa: E731
    for target in (table[:90, 1], table[::2, 0], table[0, :1].expand(90), table[:90, 2].flip(0)):
        torch._dynamo.reset()
        results = []
        for f in (torch.compile(call, fullgraph=True), call):
            a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            loss = f(a, b, target)
            results.append([loss.detach(), *torch.autograd.grad(loss.sum(), [a, b])])
        for got, want in zip(*results):
            assert torch.equal(got, want)
    leaf = x.clone().requires_grad_(True)                                # the operator by itself
    got = torch.ops.cinnamon_b200.linear_ce_fwd(leaf, w, table[:90, 1].long(), -100, 0, False)[0]
    assert torch.equal(got, call(leaf, w, table[:90, 1]))


def test_compiled_loss_refuses_operands_of_other_devices():
    from cinnamon_b200 import kernels as K
    x, w = torch.zeros(5, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(7, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(5, device="cuda", dtype=torch.int64)
    f = torch.compile(lambda x, w, t: K.linear_cross_entropy(x, w, t))
    for args in ((x, w, t.cpu()), (x, w.cpu(), t), (x.cpu(), w, t)):
        torch._dynamo.reset()
        with pytest.raises(Exception, match="Inputs must be on CUDA"):
            f(*args)
    for args in ((x, w, t.cpu()), (x, w, t[:4]), (x, w.cpu(), t)):
        with pytest.raises(AssertionError, match="linear_cross_entropy|Inputs must be on CUDA"):
            torch.ops.cinnamon_b200.linear_ce_fwd(*args, -100, 1, False)
    loss, state, sx, sw = torch.ops.cinnamon_b200.linear_ce_fwd(x, w, t, -100, 1, False)
    assert abs(float(loss) - math.log(7.0)) <= 2.0 ** -20
    with pytest.raises(AssertionError, match="left for"):
        torch.ops.cinnamon_b200.linear_ce_bwd(loss, x, w, state[:256], 1, True, True)
    with pytest.raises(AssertionError, match="left for"):
        torch.ops.cinnamon_b200.linear_ce_finish(loss, state, sx, sw, 5, 7, 64, x.dtype, 1, True, True)
    assert K.device_status() == 0


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("frozen", ["x", "weight", "neither"])
@pytest.mark.parametrize("T,d", [(150, 100), (2100, 1030)])             # (the second: a mean's gradients are made in the forward)
def test_compiled_loss_with_one_side_frozen(T, d, frozen, reduction):
    """The eager call's bits, and neither time nor memory for the gradient that nobody asked for."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(7)
    V = 40000
    x, w = torch.randn(T, d, generator=g).cuda(), (torch.randn(V, d, generator=g) * 0.1).cuda()
    target = torch.randint(0, V, (T,), generator=g).cuda()
    target[::9] = -100
    call = lambda x, w: K.linear_cross_entropy(x, w, target, reduction=reduction)      # noqa: E731
    up = torch.randn((T,) if reduction == "none" else (), generator=g).cuda()
    results, most = [], []
    for compiled in (False, True):
        torch._dynamo.reset()
        f = torch.compile(call, fullgraph=True) if compiled else call
        a, b = x.bfloat16().requires_grad_(frozen != "x"), w.bfloat16().requires_grad_(frozen != "weight")
        leaves = [t for t in (a, b) if t.requires_grad]
        torch.autograd.grad(f(a, b), leaves, up)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = f(a, b)
        results.append([loss.detach(), *torch.autograd.grad(loss, leaves, up)])
        most.append(torch.cuda.max_memory_allocated() - before)
    for got, want in zip(results[1], results[0]):
        assert got.shape == want.shape and torch.equal(got, want)
    assert most[1] <= most[0] + (4 << 20)                                # (a gradient of this weight: 8 and 82 MB)


@pytest.mark.parametrize("op", ["loss", "rotary", "route", "route_reference"])
@pytest.mark.parametrize("everything", [False, True])
def test_capture_beside_a_living_graph_of_a_leaf_behind_views(op, everything):
    """A leaf behind a transpose, a slice or a product has its node on the default stream as well: the captured backward is refused before it gets there.
    A captured forward alone, and a backward that ends in front of the leaf, go through."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(4)
    x, w = (torch.randn(40, 96, generator=g).cuda().bfloat16().requires_grad_(True) for _ in range(2))
    q = torch.randn(1, 40, 2, 64, generator=g).cuda().requires_grad_(True)
    target, positions, bias = torch.arange(40, device="cuda"), torch.arange(40, device="cuda"), torch.zeros(64, device="cuda")
    freq, _ = K.rotary_frequencies(32, device="cuda")
    shown = {"loss": lambda: (x[:, 8:72] * 2, w.narrow(1, 16, 64)), "rotary": lambda: (q.transpose(1, 2) * 1.0,),
             "route": lambda: (x[:, :64],), "route_reference": lambda: (x[:, :64],)}[op]
    calls = {"loss": lambda a, b: K.linear_cross_entropy(a, b, target), "rotary": lambda a: K.rotary(a, None, positions, freq)[0].sum(),
             "route": lambda a: K.moe_route(a, bias, 2, scores="softmax")["top_gates"].sum(), "route_reference": lambda a: K.moe_route(a, bias, 2)["top_gates"].sum()}
    call = lambda: calls[op](*shown())                                   # noqa: E731
    leaves = [q] if op == "rotary" else [x] if op.startswith("route") else [x, w]

    def back(loss):
        if not everything:
            return torch.autograd.grad(loss, leaves)
        loss.backward()
        return [t.grad for t in leaves]
    earlier = call()
    want = torch.autograd.grad(earlier, leaves, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with pytest.raises(AssertionError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                back(call())
        forward, inner = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(forward, stream=side):
            loss = call().detach()
        with torch.cuda.graph(inner, stream=side):
            parts = shown()
            between = torch.autograd.grad(calls[op](*parts), parts)
        del earlier, parts
        gc.collect()                                                     # (the refused step's graph, in its exception's frames)
        for t in leaves:
            t.grad = None
        torch.autograd.grad(call(), leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = back(call())
    torch.cuda.current_stream().wait_stream(side)
    for g in (forward, inner, graph):
        g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(loss, call().detach()) and all(t.abs().sum() > 0 for t in between)
    assert K.device_status() == 0


@pytest.mark.parametrize("frozen", [0, 1, None])
def test_compiled_rotary_with_one_side_frozen(frozen):
    """The eager call's bits, and no gradient for the side that takes none (heads of other lengths: `start` counts from each one's end)."""
    from cinnamon_b200 import kernels as K
    g = torch.Generator().manual_seed(8)
    q, k = torch.randn(2, 8, 600, 96, generator=g).bfloat16().cuda(), torch.randn(2, 4, 600, 160, generator=g).bfloat16().cuda()
    freq, positions = K.rotary_frequencies(32, device="cuda")[0], torch.arange(600, device="cuda")
    call = lambda q, k: K.rotary(q, k, positions, freq, start=-32)       # noqa: E731
    results, most = [], []
    for compiled in (False, True):
        torch._dynamo.reset()
        f = torch.compile(call, fullgraph=True) if compiled else call
        a, b = (t.clone().requires_grad_(i != frozen) for i, t in enumerate((q, k)))
        leaves = [t for t in (a, b) if t.requires_grad]
        torch.autograd.grad(f(a, b), leaves, [q, k])
        out = f(a, b)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = torch.autograd.grad(out, leaves, [q, k])
        most.append(torch.cuda.max_memory_allocated() - before)
        results.append([*(t.detach() for t in out), *grads])
    for got, want in zip(results[1], results[0]):
        assert got.shape == want.shape and torch.equal(got, want)
    assert most[1] <= most[0] + (1 << 20)                                # (a gradient of these: 1.8 and 1.5 MB)
