"""``linear_cross_entropy`` against the formula in 64 bits on the same 16-bit operands.

Tolerances, per element, from the arithmetic (u: half a step of the operands' type, 2^-8 for bf16 and 2^-11 for fp16):
  logits   fp32 sums of exact products: ez = (d / 16 + 8) 2^-22 max_v sum_k |x_k w_vk| (sixteen products a step; a step may truncate)
  loss     2 ez, the exponentials' and the sum's 2^-20, and 2^-22 of the loss and of the maximum
  dz       rounded once to the operands' type: u |dz|, and the probabilities' own 2 ez + 2^-20; made early (sums and means over 2048
           rows or more of 1024 or more) from exponentials in fp16: 2^-11 of the probability more, and 2^-25 of the largest one beside it;
           for up to 128 rows held in two parts: u^2 |dz| in place of u |dz|
  dx, dW   the errors of dz through the product, fp32 sums (their number of terms / 16 + 8) 2^-22 of the sum of absolute terms, and one
           rounding of the result, u |dx| (in fp16 at least half the smallest step, 2^-25)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _inputs(T, V, d, dtype, seed=0, ignored=0.0, lift=6.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, d, generator=g) * (0.5 / math.sqrt(d))).to(dtype)
    target = torch.randint(0, V, (T,), generator=g)
    hit = w[target].float()
    x = torch.randn(T, d, generator=g) + lift * torch.rand(T, 1, generator=g) * hit / hit.pow(2).sum(-1, keepdim=True).clamp(min=0.05)
    if ignored:
        target[torch.rand(T, generator=g) < ignored] = -100
    return x.to(dtype).cuda(), w.cuda(), target.cuda()


def _oracle(x, w, target, grad, ignore=-100, early=False, few=False):
    """Losses, gradients and the tolerances of all three, in 64 bits.  ``grad``: the gradient of every token's loss."""
    u = HALF_STEP[x.dtype]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    V, d = w.shape
    use = (target != ignore) & (target >= 0) & (target < V)
    rows = torch.nonzero(use)[:, 0]
    xr, wd, t = x[rows].double(), w.double(), target[rows].long()
    z = xr @ wd.t()
    ez = (d / 16 + 8) * 2.0 ** -22 * (xr.abs() @ wd.abs().t()).amax(-1, keepdim=True) if len(rows) else z.new_zeros(0, 1)
    lse = torch.logsumexp(z, -1, keepdim=True)
    at = torch.arange(len(rows), device=x.device)
    loss = torch.zeros(len(x), dtype=torch.float64, device=x.device)
    loss_tol = torch.zeros_like(loss)
    loss[rows] = lse[:, 0] - z[at, t]
    if len(rows):
        loss_tol[rows] = 2 * ez[:, 0] + 2.0 ** -20 + 2.0 ** -22 * (loss[rows].abs() + z.abs().amax(-1))
    p = torch.exp(z - lse)
    dz = p.clone()
    dz[at, t] -= 1.0
    gr = grad[rows].double()[:, None]
    # dz is held relative to the largest gradient, in fp16 times 2^14
    held = (2.0 ** -39 if x.dtype == torch.float16 else 0.0) * (gr.abs().amax() if len(rows) else 0.0)
    e_dz = ((u * u if few else u) * dz.abs() + (1 + u) * p * (2 * ez + 2.0 ** -20)) * gr.abs() + held + 2.0 ** -22 * (dz * gr).abs()
    if early:
        e_dz = e_dz + (1 + u) * (2.0 ** -11 * p + 2.0 ** -25) * gr.abs()
    dz = dz * gr
    dx, dx_tol = torch.zeros(len(x), d, dtype=torch.float64, device=x.device), torch.zeros(len(x), d, dtype=torch.float64, device=x.device)
    dx[rows] = dz @ wd
    dx_tol[rows] = (e_dz + (V / 16 + 8) * 2.0 ** -22 * dz.abs()) @ wd.abs() * (1 + u) + u * dx[rows].abs() + tiny
    dw = dz.t() @ xr
    dw_tol = (e_dz + (len(rows) / 16 + 8) * 2.0 ** -22 * dz.abs()).t() @ xr.abs() * (1 + u) + u * dw.abs() + tiny
    return loss, loss_tol, dx, dx_tol, dw, dw_tol


def _within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() - tol).max() if got.numel() else torch.tensor(-1.0)
    assert over <= 0, f"{what}: {float(over):.3g} over the tolerance at {int(((got - want).abs() - tol).argmax())}"


def _run(x, w, target, grad=None, reduction="mean", **kw):
    from cinnamon_b200 import kernels as K
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = K.linear_cross_entropy(x, w, target, reduction=reduction, **kw)
    assert loss.dtype == torch.float32
    gx, gw = torch.autograd.grad(loss, [x, w], grad if grad is not None else torch.ones_like(loss))
    assert gx.dtype == x.dtype and gw.dtype == w.dtype
    assert K.device_status() == 0
    return loss.detach(), gx, gw


SHAPES = [
    (1, 1, 8, 0.0), (1, 2, 8, 0.0), (1, 1000, 64, 0.0), (2, 257, 72, 0.0), (7, 255, 64, 0.0), (64, 5003, 128, 0.0), (129, 256, 64, 0.0),
    (130, 513, 520, 0.3), (256, 8, 64, 0.0), (257, 33, 16, 0.5), (300, 1000, 1032, 0.0), (1023, 300, 64, 0.2), (1025, 777, 136, 0.9),
    (2100, 2050, 264, 0.4), (4097, 64, 40, 0.1), (2049, 300, 1024, 0.0), (4500, 515, 1032, 0.6), (2300, 70, 2056, 0.1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,d,ignored", SHAPES)
def test_mean_loss_and_gradients(T, V, d, ignored, dtype):
    x, w, target = _inputs(T, V, d, dtype, seed=T + V, ignored=ignored)
    target[0] = V - 1                                                  # (some token counts, and the last word is hit)
    n = int((target != -100).sum())
    up = 64.0
    want = _oracle(x, w, target, torch.full((T,), up / n, device="cuda"), early=T >= 2048 and d >= 1024)
    loss, gx, gw = _run(x, w, target, torch.tensor(up, device="cuda"))
    _within(loss, want[0].sum() / n, want[1].sum() / n + 2.0 ** -23 * want[0].sum() / n, "loss")
    _within(gx, want[2], want[3], "grad_x")
    _within(gw, want[4], want[5], "grad_w")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,d,ignored", [(1, 300, 64, 0.0), (33, 70, 24, 0.3), (515, 1111, 200, 0.5)])
def test_losses_of_tokens_with_a_gradient_each(T, V, d, ignored, dtype):
    x, w, target = _inputs(T, V, d, dtype, seed=3 * T, ignored=ignored)
    target[T // 2] = 0
    grad = torch.randn(T, generator=torch.Generator().manual_seed(T)).cuda() * 3
    grad[T // 3] = 0.0
    want = _oracle(x, w, target, grad)
    loss, gx, gw = _run(x, w, target, grad, reduction="none")
    _within(loss, want[0], want[1], "loss")
    assert (loss[target == -100] == 0).all()
    _within(gx, want[2], want[3], "grad_x")
    _within(gw, want[4], want[5], "grad_w")
    total, sx, sw = _run(x, w, target, torch.tensor(2.0, device="cuda"), reduction="sum")
    want = _oracle(x, w, target, torch.full((T,), 2.0, device="cuda"))
    _within(total, want[0].sum(), want[1].sum() + 2.0 ** -23 * want[0].sum(), "sum")
    _within(sx, want[2], want[3], "grad_x of the sum")
    _within(sw, want[4], want[5], "grad_w of the sum")


@pytest.mark.parametrize("early", [False, True])
def test_in_pieces(early):
    """More than one piece: of the vocabulary (512 MiB of the logits' gradient), where dx is added up over them, or early of the
    tokens (1.25 GiB), where dW is."""
    T, V, d = (90000 if early else 65536) + 130, 8192 + 70, 1024 if early else 64
    x, w, target = _inputs(T, V, d, torch.bfloat16, seed=5, ignored=0.01)
    grad = torch.full((T,), 1.0, device="cuda")
    n = int((target != -100).sum()) if early else 1.0
    loss, gx, gw = _run(x, w, target) if early else _run(x, w, target, grad, reduction="none")
    for at in (0, T - 2048):
        want = _oracle(x[at:at + 2048], w, target[at:at + 2048], grad[:2048] / n, early=early)
        _within(gx[at:at + 2048], want[2], want[3], "grad_x")
        if not early:
            _within(loss[at:at + 2048], want[0], want[1], "loss")
    # the weight's gradient and the mean, from the whole batch in pieces of rows
    dw, tol, total, total_tol = 0.0, 0.0, 0.0, 0.0
    for at in range(0, T, 8192):
        part = _oracle(x[at:at + 8192], w, target[at:at + 8192], grad[at:at + 8192] / n, early=early)
        dw, tol, total, total_tol = dw + part[4], tol + part[5], total + part[0].sum(), total_tol + part[1].sum()
    _within(gw, dw, tol + (T / 16) * 2.0 ** -22 * tol / HALF_STEP[torch.bfloat16], "grad_w")
    if early:
        _within(loss, total / n, total_tol / n + 2.0 ** -23 * total / n, "loss")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_early_gradients_alone_twice_and_late(dtype):
    """Sums over many tokens: each gradient by itself, a backward that is run again, another scale of the loss, and the late way's result."""
    from cinnamon_b200 import kernels as K
    T, V, d = 2300, 1030, 1032
    x, w, target = _inputs(T, V, d, dtype, seed=T, ignored=0.25)
    assert K._host.linear_ce_early(T, V, d, 2, 0) == 1 and K._host.linear_ce_early(T, V, d, 0, 0) == 0
    want = _oracle(x, w, target, torch.full((T,), 3.0, device="cuda"), early=True)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = K.linear_cross_entropy(a, b, target, reduction="sum")
    three = torch.tensor(3.0, device="cuda")
    first = torch.autograd.grad(loss, [a, b], three, retain_graph=True)
    _within(loss.detach(), want[0].sum(), want[1].sum() + 2.0 ** -23 * want[0].sum(), "sum")
    _within(first[0], want[2], want[3], "grad_x")
    _within(first[1], want[4], want[5], "grad_w")
    first[0].zero_()                                                   # (what was returned is the caller's)
    again = torch.autograd.grad(loss, [a, b], three, retain_graph=True)
    _within(again[0], want[2], want[3], "grad_x again")
    assert torch.equal(again[1], first[1])
    assert torch.equal(torch.autograd.grad(K.linear_cross_entropy(a, w, target, reduction="sum"), a, three)[0], again[0])
    assert torch.equal(torch.autograd.grad(K.linear_cross_entropy(x, b, target, reduction="sum"), b, three)[0], again[1])
    late = _run(x, w, target, torch.full((T,), 3.0, device="cuda"), reduction="none")
    u = HALF_STEP[dtype]
    for e, l in zip(again, late[1:]):
        assert (e.float() - l.float()).norm() <= 4 * u * l.float().norm()
    # in place after the forward: the gradients are those of the values it was called with
    loss = K.linear_cross_entropy(a, b, target, reduction="sum")
    with torch.no_grad():
        assert K.linear_cross_entropy(a, b, target, reduction="sum") == loss


@pytest.mark.parametrize("T,d", [(256, 64), (2304, 1024)])
def test_well_predicted_tokens_keep_their_gradient(T, d):
    """Targets with probabilities up to 1 - 1e-5: what is left of 1 - p has to come through."""
    V = 500
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(V, d, generator=g) * (8 / math.sqrt(d))).bfloat16().cuda()
    target = torch.randint(0, V, (T,), generator=g).cuda()
    x = (w[target].float() * torch.linspace(0.05, 0.6, T, device="cuda")[:, None]).bfloat16()
    early = T >= 2048
    want = _oracle(x, w, target, torch.full((T,), 1.0, device="cuda"), early=early)
    loss, gx, gw = _run(x, w, target, reduction="sum") if early else _run(x, w, target, torch.ones(T, device="cuda"), reduction="none")
    if not early:
        _within(loss, want[0], want[1], "loss")
    _within(gx, want[2], want[3], "grad_x")


@pytest.mark.parametrize("T,d", [(700, 96), (2500, 1040), (5000, 1040)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_ignored_rows_reach_nothing(reduction, T, d):
    V = 999
    x, w, target = _inputs(T, V, d, torch.bfloat16, seed=11, ignored=0.4)
    grad = torch.randn(T, device="cuda") if reduction == "none" else torch.tensor(1.0, device="cuda")
    clean = _run(x, w, target, grad, reduction=reduction)
    x2 = x.clone()
    bad = torch.nonzero(target == -100)[:, 0]
    x2[bad[0::3]], x2[bad[1::3]], x2[bad[2::3]] = float("nan"), float("inf"), float("-inf")
    if reduction == "none":
        grad = grad.clone()
        grad[bad] = float("nan")
    dirty = _run(x2, w, target, grad, reduction=reduction)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert (dirty[1][bad] == 0).all()


@pytest.mark.parametrize("T", [300, 2500])
def test_nothing_but_ignored_rows(T):
    x, w, _ = _inputs(T, 400, 64 if T < 2048 else 1024, torch.bfloat16)
    target = torch.full((T,), -100, device="cuda")
    loss, gx, gw = _run(x, w, target)
    assert torch.isnan(loss) and (gx == 0).all() and (gw == 0).all()
    loss, gx, gw = _run(x, w, target, reduction="sum")
    assert loss == 0 and (gx == 0).all() and (gw == 0).all()
    loss, gx, gw = _run(x, w, target, reduction="none")
    assert (loss == 0).all() and (gx == 0).all() and (gw == 0).all()


def test_no_rows():
    from cinnamon_b200 import kernels as K
    w = torch.randn(100, 64, device="cuda", dtype=torch.bfloat16)
    x, target = w[:0], torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, gx, gw = _run(x, w, target)
    assert torch.isnan(loss) and gx.shape == (0, 64) and (gw == 0).all()
    assert _run(x, w, target, reduction="sum")[0] == 0
    assert K.linear_cross_entropy(x, w, target, reduction="none").shape == (0,)


@pytest.mark.parametrize("T", [200, 4500])
def test_targets_that_are_no_words(T):
    V, d = 300, 64 if T < 2048 else 1024
    x, w, target = _inputs(T, V, d, torch.bfloat16, seed=2)
    bad = target.clone()
    bad[3], bad[77], bad[150] = V, -1, 1 << 40
    loss, gx, gw = _run(x, w, bad, torch.ones(T, device="cuda"), reduction="none")
    out = torch.tensor([3, 77, 150], device="cuda")
    assert torch.isnan(loss[out]).all() and (gx[out] == 0).all() and int(torch.isnan(loss).sum()) == 3
    without = target.clone()
    without[out] = -100
    same = _run(x, w, without, torch.ones(T, device="cuda"), reduction="none")
    assert torch.equal(gx, same[1]) and torch.equal(gw, same[2])
    assert torch.isnan(_run(x, w, bad)[0])


def test_another_ignored_index_and_a_word_of_that_name():
    x, w, target = _inputs(150, 40, 64, torch.bfloat16, seed=8)
    loss, gx, _ = _run(x, w, target, torch.ones(150, device="cuda"), reduction="none", ignore_index=7)
    assert (loss[target == 7] == 0).all() and (gx[target == 7] == 0).all() and (loss[target != 7] > 0).all()


@pytest.mark.parametrize("d", [1, 3, 63, 100])
def test_odd_rows_and_strides(d):
    """Row lengths, pitches and bases that the copies cannot read in place."""
    T, V = 190, 333
    x, w, target = _inputs(T, V, d + 5, torch.bfloat16, seed=d)
    xs, ws = x[:, 2:2 + d], w[:, 3:3 + d]
    n = T
    want = _oracle(xs, ws, target, torch.full((T,), 1.0 / n, device="cuda"))
    loss, gx, gw = _run(xs, ws, target)
    _within(gx, want[2], want[3], "grad_x")
    _within(gw, want[4], want[5], "grad_w")
    same = _run(xs.contiguous(), ws.contiguous(), target)
    for a, b in zip((loss, gx, gw), same):
        assert torch.equal(a, b)


def test_batches_transposed_views_and_int32_targets():
    B, L, V, d = 5, 37, 301, 64
    x, w, target = _inputs(B * L, V, d, torch.bfloat16, seed=4, ignored=0.2)
    flat = _run(x, w, target)
    shaped = _run(x.view(B, L, d), w, target.view(B, L).int())
    assert torch.equal(shaped[0], flat[0]) and torch.equal(shaped[1].view(-1, d), flat[1]) and torch.equal(shaped[2], flat[2])
    turned = _run(x.view(B, L, d).transpose(0, 1), w, target.view(B, L).t())
    assert torch.equal(turned[1].transpose(0, 1).reshape(-1, d), flat[1])
    wt = _run(x, w.t().contiguous().t(), target)
    assert torch.equal(wt[1], flat[1]) and torch.equal(wt[2], flat[2])
    one = _run(x[0], w, target[0], reduction="none") if target[0] != -100 else None
    assert one is None or one[0].shape == ()
    wide = x[:1].expand(B, d)
    t = torch.arange(B, device="cuda")
    assert torch.equal(_run(wide, w, t)[2], _run(wide.contiguous(), w, t)[2])


def test_gradients_one_at_a_time_and_none():
    from cinnamon_b200 import kernels as K
    x, w, target = _inputs(140, 600, 64, torch.bfloat16, seed=6)
    loss, gx, gw = _run(x, w, target)
    a = x.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(K.linear_cross_entropy(a, w, target), a)[0], gx)
    b = w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(K.linear_cross_entropy(x, b, target), b)[0], gw)
    plain = K.linear_cross_entropy(x, w, target)
    assert not plain.requires_grad and torch.equal(plain, loss)


def test_the_same_bits_every_time():
    x, w, target = _inputs(3000, 4001, 264, torch.bfloat16, seed=9, ignored=0.3)
    first = _run(x, w, target)
    for _ in range(3):
        for a, b in zip(first, _run(x, w, target)):
            assert torch.equal(a, b)


def test_autocast_as_for_a_linear():
    """fp32 activations and master weights: cast as F.linear casts them, gradients of the parameters' type."""
    from cinnamon_b200 import kernels as K
    x, w, target = _inputs(130, 400, 64, torch.bfloat16, seed=12)
    ref = _run(x, w, target)
    xf, wf = x.float().requires_grad_(True), w.float().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = K.linear_cross_entropy(xf, wf, target)
    gx, gw = torch.autograd.grad(loss, [xf, wf])
    assert gx.dtype == gw.dtype == torch.float32
    assert torch.equal(loss, ref[0]) and torch.equal(gx, ref[1].float()) and torch.equal(gw, ref[2].float())


def test_gradient_against_differences():
    """Central differences of the summed loss along directions on the operands' grid.  With steps s of the logits' change in
    [-a, a] the third derivative of a token's log-sum-exp along the direction is below a^3 (a distribution's third central moment on an
    interval of width 2 a is at most 4 a^3 / (3 sqrt 3)), so the difference is off by at most T a^3 / 6 and by the losses' own error."""
    T, V, d = 40, 200, 64
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-16, 17, (T, d), generator=g).float() / 16
    w = torch.randint(-16, 17, (V, d), generator=g).float() / 64
    target = torch.randint(0, V, (T,), generator=g).cuda()
    hx = torch.randint(-1, 2, (T, d), generator=g).float() / 32
    hw = torch.randint(-1, 2, (V, d), generator=g).float() / 128
    from cinnamon_b200 import kernels as K
    f = lambda a, b: float(K.linear_cross_entropy(a.bfloat16().cuda(), b.bfloat16().cuda(), target, reduction="sum"))      # noqa: E731
    _, gx, gw = _run(x.bfloat16().cuda(), w.bfloat16().cuda(), target, reduction="sum")
    loss, loss_tol, dx, dx_tol, dw, dw_tol = _oracle(x.bfloat16().cuda(), w.bfloat16().cuda(), target, torch.ones(T, device="cuda"))
    for h, at, moved, tol in ((hx, gx, (hx @ w.t()), dx_tol), (hw, gw, (x @ hw.t()), dw_tol)):
        a = float(moved.abs().max())
        diff = (f(x + h, w) - f(x - h, w)) / 2 if h is hx else (f(x, w + h) - f(x, w - h)) / 2
        slack = T * a ** 3 / 6 + float(loss_tol.sum()) * 2 + float((tol.cpu() * h.abs()).sum())
        assert abs(diff - float((at.float().cpu() * h).sum())) <= slack
        assert slack < 0.2 * abs(diff) or abs(diff) < 1.0


@pytest.mark.parametrize("T", [400, 2400])
def test_other_streams_and_a_captured_step(T):
    from cinnamon_b200 import kernels as K
    d = 128 if T < 2048 else 1024
    x, w, target = _inputs(T, 1500, d, torch.bfloat16, seed=21, ignored=0.2)
    ref = _run(x, w, target)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _run(x, w, target)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(ref, other):
        assert torch.equal(a, b)
    xs, ws, ts = x.clone().requires_grad_(True), w.clone().requires_grad_(True), target.clone()
    graphs = []
    for _ in range(2):                                                 # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            torch.autograd.grad(K.linear_cross_entropy(xs, ws, ts), [xs, ws])
            with torch.cuda.graph(graph, stream=side):
                loss = K.linear_cross_entropy(xs, ws, ts)
                gx, gw = torch.autograd.grad(loss, [xs, ws])
        graphs.append((graph, loss, gx, gw))
    x2, w2, t2 = _inputs(T, 1500, d, torch.bfloat16, seed=22, ignored=0.6)
    want = _run(x2, w2, t2)
    with torch.no_grad():
        xs.copy_(x2), ws.copy_(w2), ts.copy_(t2)
    torch.cuda.synchronize()
    for graph, loss, gx, gw in graphs * 2:
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((loss.detach(), gx, gw), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [600, 2600])
def test_a_cap_on_the_sms_changes_no_bits(T):
    from cinnamon_b200 import kernels as K
    x, w, target = _inputs(T, 2000, 128 if T < 2048 else 1024, torch.bfloat16, seed=31)
    ref = _run(x, w, target)
    try:
        for cap in (1, 2, 37):
            K.set_gemm_sm_limit(cap)
            for a, b in zip(ref, _run(x, w, target)):
                assert torch.equal(a, b)
    finally:
        K.set_gemm_sm_limit(0)


def test_refusals():
    from cinnamon_b200 import kernels as K
    x, w, target = _inputs(10, 20, 64, torch.bfloat16)
    call = K.linear_cross_entropy
    for bad, what in [((x.float(), w.float(), target), "16-bit"), ((x, w.half(), target), "16-bit"), ((x, w[:, :32], target), "vocabulary"),
                      ((x, w, target[:5]), "one entry"), ((x, w, target.float()), "int64"), ((x, w.cpu(), target), "CUDA"),
                      ((x, w[:0], target), "empty")]:
        with pytest.raises(AssertionError, match=what):
            call(*bad)
    with pytest.raises(AssertionError, match="reduction"):
        call(x, w, target, reduction="avg")
    a = x.detach().requires_grad_(True)
    with pytest.raises(AssertionError, match="second derivative"):
        torch.autograd.grad(call(a, w, target), a, create_graph=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("T,V,d,ignored", [(1, 700, 64, 0.0), (2, 33, 200, 0.0), (3, 1000, 512, 0.3), (31, 300, 72, 0.0), (32, 300, 72, 0.5), (33, 2000, 256, 0.0),
                                           (64, 513, 128, 0.0), (65, 513, 128, 0.4), (127, 4000, 64, 0.2), (128, 260, 1032, 0.0), (128, 32000, 512, 0.9)])
def test_a_few_tokens_lose_nothing_to_dz(T, V, d, ignored, reduction, dtype):
    """One token's dz is a factor of all that it adds: its rounding would not average out."""
    x, w, target = _inputs(T, V, d, dtype, seed=T + V, ignored=ignored, lift=14.0)
    target[0] = V // 2
    n = int((target >= 0).sum())
    grad = torch.randn(T, generator=torch.Generator().manual_seed(5)).cuda() if reduction == "none" else None
    loss, gx, gw = _run(x, w, target, grad, reduction)
    per = grad if reduction == "none" else torch.full((T,), 1.0 / n, device="cuda")
    _, _, dx, dx_tol, dw, dw_tol = _oracle(x, w, target, per, few=True)
    _within(gx, dx, dx_tol, "dx")
    _within(gw, dw, dw_tol, "dw")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,ignored", [(40, 0.0), (300, 0.3), (2300, 0.1)])
def test_infinite_gradients_are_their_own_tokens(T, ignored, dtype):
    """One token's infinite or NaN gradient leaves the others' rows as they are."""
    x, w, target = _inputs(T, 500, 136, dtype, seed=T, ignored=ignored)
    bad = torch.tensor([5, 9, 17], device="cuda")
    target[bad] = 3
    others = torch.ones(T, dtype=torch.bool, device="cuda")
    others[bad] = False
    grad = torch.randn(T, generator=torch.Generator().manual_seed(1)).cuda()
    for rest in (grad, torch.zeros_like(grad)):
        clean, dirty = rest.clone(), rest.clone()
        clean[bad] = 0.0
        dirty[5], dirty[9], dirty[17] = float("inf"), float("nan"), float("-inf")
        want, got = _run(x, w, target, clean, reduction="none"), _run(x, w, target, dirty, reduction="none")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][others], want[1][others])
        assert not torch.isfinite(got[1][bad]).any() and not torch.isfinite(got[2]).any()
        if ignored:                                                    # (an ignored token's gradient is nobody's)
            dirty = clean.clone()
            dirty[target == -100] = float("inf")
            assert all(torch.equal(a, b) for a, b in zip(_run(x, w, target, dirty, reduction="none"), want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,d", [(2304, 512, 1024), (2050, 500, 1040)])
def test_rare_words_beside_a_likely_one(T, V, d, dtype):
    """Gradients made in the forward: rows of dW of words that are 8 to 24 nats less likely than the best of their 128 neighbours, each against its
    own size.  The exponentials are held in fp16 relative to that best one, times 2^15: an error of 2^-11 of each, and at least 2^-40 of the best one
    (half of fp16's smallest step, 2^-25)."""
    from cinnamon_b200 import kernels as K
    assert K._host.linear_ce_early(T, V, d, 2, 0) == 1
    g = torch.Generator().manual_seed(V)
    u = HALF_STEP[dtype]
    along = torch.full((d,), d ** -0.5)
    x = (8 * along + 0.3 * torch.randn(T, d, generator=g)).to(dtype).cuda()
    less = 8 + 16 * torch.rand(V, generator=g)
    less[::128] = torch.arange((V + 127) // 128).float()                # the likely ones, one in 128
    w = (-less[:, None] / 8 * along + 0.02 * torch.randn(V, d, generator=g)).to(dtype).cuda()
    target = (torch.randint(0, (V + 127) // 128, (T,), generator=g) * 128).cuda()
    target[7::50] = -100
    grad = torch.ones(T, device="cuda")
    _, _, dx, dx_tol, dw, dw_tol = _oracle(x, w, target, grad)
    use = target >= 0
    p = torch.softmax(x[use].double() @ w.double().t(), -1)
    best = torch.nn.functional.pad(p, (0, -V % 128)).unflatten(1, (-1, 128)).amax(-1).repeat_interleave(128, 1)[:, :V]
    e = (1 + u) * (2.0 ** -11 * p + 2.0 ** -40 * best)
    dw_tol = dw_tol + e.t() @ x[use].double().abs() * (1 + u)
    dx_tol[use] += e @ w.double().abs() * (1 + u)
    _, gx, gw = _run(x, w, target, reduction="sum")
    _within(gx, dx, dx_tol, "grad_x")
    _within(gw, dw, dw_tol, "grad_w")
    rare = (less > 17) & (less < 20)
    assert rare.sum() > 20 and (dw_tol[rare].norm(dim=1) <= 0.1 * dw[rare].norm(dim=1)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,d", [(200, 300, 7168), (70, 5000, 1040), (300, 300, 64)])
def test_sums_that_lose_nothing(T, V, d, dtype):
    """Sixteen non-zeros on a coarse grid in each row: the tensor cores' sums are exact, and the factor of 1 + 0.3 d / 16 2^-24 that makes good for what
    such sums lose on average is itself the error, of that much of the largest logit; beside it the exponentials' 2^-20 and the fp32 of
    logits and loss, 2^-22."""
    g = torch.Generator().manual_seed(d)
    at = torch.arange(16) * (d // 16) + 3
    x, w = torch.zeros(T, d), torch.zeros(V, d)
    x[:, at] = torch.randint(-8, 9, (T, 16), generator=g).float() / 4
    w[:, at] = torch.randint(-16, 17, (V, 16), generator=g).float() / 8
    x, w, target = x.to(dtype).cuda(), w.to(dtype).cuda(), torch.randint(0, V, (T,), generator=g).cuda()
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, -1) - z.gather(1, target[:, None])[:, 0]
    tol = 0.3 * (d // 16) * 2.0 ** -24 * z.abs().amax(-1) + 2.0 ** -20 + 2.0 ** -22 * (want + z.abs().amax(-1))
    assert z.max() > 10
    loss, _, _ = _run(x, w, target, torch.ones(T, device="cuda"), reduction="none")
    _within(loss, want, tol, "loss")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_operands_changed_in_place_after_the_forward(dtype):
    """Gradients made in the forward are those of the values it was called with, whatever the operands and targets hold by the time of the backward; made in the
    backward, they are refused."""
    from cinnamon_b200 import kernels as K
    T, V, d = 2300, 700, 1032
    x, w, target = _inputs(T, V, d, dtype, seed=77, ignored=0.2)
    want = _run(x, w, target, reduction="sum")
    for side in (None, 0, 1):                                            # (a frozen one too)
        a, b, t = x.clone().requires_grad_(side != 0), w.clone().requires_grad_(side != 1), target.clone()
        leaves = [v for v in (a, b) if v.requires_grad]
        loss = K.linear_cross_entropy(a, b, t, reduction="sum")
        with torch.no_grad():
            a.normal_(), b.zero_(), t.fill_(1)
        got = torch.autograd.grad(loss, leaves)
        assert torch.equal(loss.detach(), want[0])
        for v, g in zip(got, [want[1 + i] for i in range(2) if i != side]):
            assert torch.equal(v, g)
    up = torch.ones(T, device="cuda")
    want = _run(x, w, target, up, reduction="none")
    for changed in range(3):
        a, b, t = x.clone().requires_grad_(True), w.clone().requires_grad_(True), target.clone()
        loss = K.linear_cross_entropy(a, b, t, reduction="none")
        with torch.no_grad():
            (a, b, t)[changed].zero_()
        if changed == 2:                                                 # (the backward reads its own copy of the targets)
            assert torch.equal(torch.autograd.grad(loss, a, up)[0], want[1])
            continue
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, [a, b], up)
