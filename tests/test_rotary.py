"""``rotary`` against the formula in 64 bits.

Tolerance: cosine and sine are within 2^-21 (sincospif's two last bits, the angle's rounding within an eighth of a turn, the
magnitude's product), and the position's angle is off by its frequency's rounding, position x frequency x 2^-51; products and
their sum in fp32 add 2^-23 of |a| + |b|; the result is rounded once, half a step of its type."""
import math

import pytest
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _oracle(t, positions, freq, interleaved, start, magnitude, inverse=False):
    x = t.double().cpu()
    n = freq.numel()
    at = start if start >= 0 else x.shape[-1] + start
    angle = positions.cpu().double()[..., None] * freq.cpu().double()
    angle = angle.expand(x.shape[0], *angle.shape[-2:])[:, None] if angle.dim() == 2 else angle[:, None]
    if inverse:
        angle = -angle
    part = x[..., at:at + 2 * n]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    ra, rb = a * c - b * s, b * c + a * s
    size = (a.abs() + b.abs()) * magnitude
    tol = size * (2.0 ** -21 + 2.0 ** -22 + angle.abs() * 2.0 ** -51)
    y, e = x.clone(), torch.zeros_like(x)
    u = HALF_STEP[t.dtype]
    tiny = 2.0 ** -25 if t.dtype == torch.float16 else 0.0
    if interleaved:
        y[..., at:at + 2 * n], e[..., at:at + 2 * n] = torch.stack([ra, rb], -1).flatten(-2), torch.stack([tol, tol], -1).flatten(-2)
    else:
        y[..., at:at + 2 * n], e[..., at:at + 2 * n] = torch.cat([ra, rb], -1), torch.cat([tol, tol], -1)
    e[..., at:at + 2 * n] += u * y[..., at:at + 2 * n].abs() + u * e[..., at:at + 2 * n] + tiny
    return y, e


def _check(got, t, *form, **kw):
    want, tol = _oracle(t, *form, **kw)
    assert got.shape == t.shape and got.dtype == t.dtype
    over = (got.double().cpu() - want).abs() - tol
    assert not got.numel() or over.max() <= 0, f"{float(over.max()):.3g} over the tolerance at {int(over.argmax())}"


def _heads(B, H, L, d, dtype, seed, first=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, H, d, generator=g).to(dtype).cuda()
    return x.transpose(1, 2) if first else x.transpose(1, 2).contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_frequency_that_is_no_number_reaches_its_pair_alone(dtype):
    from cinnamon_b200 import kernels as K
    q = _heads(1, 2, 3, 72, dtype, 5)
    freq, _ = K.rotary_frequencies(32, device="cuda")
    freq[3], freq[7] = float("nan"), float("inf")
    out, _ = K.rotary(q, None, torch.arange(3, device="cuda"), freq, interleaved=True, start=8)
    nan = torch.isnan(out)[0].all(0).all(0).cpu()
    assert nan.tolist() == [i in (14, 15, 22, 23) for i in range(72)] and torch.isnan(out).sum() == 2 * 3 * 4


# batch, heads of q and k, positions, elements of q and k, rotated, start
SHAPES = [
    (1, 1, 1, 1, 2, 2, 2, 0), (2, 3, 1, 5, 64, 64, 64, 0), (1, 8, 8, 130, 192, 192, 64, -64), (3, 7, 2, 33, 96, 40, 32, 8),
    (2, 128, 1, 3, 192, 576, 64, -64), (1, 5, 5, 17, 35, 35, 10, 3), (2, 4, 4, 9, 128, 128, 128, 0), (65, 2, 1, 1, 64, 64, 16, -16),
    (1, 2, 1, 600, 66, 66, 66, 0), (1, 1, 1, 40, 4500, 4100, 4096, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,L,d,dk,rot,start", SHAPES)
def test_both_directions(B, H, Hk, L, d, dk, rot, start, dtype, interleaved):
    from cinnamon_b200 import kernels as K
    seq_first = (B + L) % 2 == 0
    q, k = _heads(B, H, L, d, dtype, 1, seq_first).requires_grad_(True), _heads(B, Hk, L, dk, dtype, 2, seq_first).requires_grad_(True)
    freq, _ = K.rotary_frequencies(rot, device="cuda")
    positions = torch.arange(L, device="cuda") * 3 + 11
    if B > 1:
        positions = positions + 977 * torch.arange(B, device="cuda")[:, None]
    form = (positions, freq, interleaved, start, 1.25)
    oq, ok = K.rotary(q, k, *form)
    assert oq.stride() == q.stride() or q.shape[2] == 1 or q.shape[1] == 1
    _check(oq.detach(), q.detach(), *form)
    _check(ok.detach(), k.detach(), *form)
    gq, gk = _heads(B, H, L, d, dtype, 3), _heads(B, Hk, L, dk, dtype, 4)
    dq, dk_ = torch.autograd.grad([oq, ok], [q, k], [gq, gk])
    _check(dq, gq, *form, inverse=True)
    _check(dk_, gk, *form, inverse=True)
    with torch.no_grad():
        assert torch.equal(K.rotary(q, k, *form)[0], oq) and torch.equal(K.rotary(k, None, *form)[0], ok)
        a, b = q.detach().clone(), k.detach().clone()
        version = a._version
        ra, rb = K.rotary_(a, b, *form)
        assert ra is a and rb is b and a._version > version
        assert torch.equal(a, oq) and torch.equal(b, ok)


@pytest.mark.gpu
def test_far_and_negative_positions():
    from cinnamon_b200 import kernels as K
    freq, _ = K.rotary_frequencies(64, device="cuda")
    positions = torch.tensor([0, 1, -1, 4095, 65537, 1000003, -1000003, 10 ** 7 + 19, 2 ** 24 + 1], device="cuda")
    q = _heads(1, 2, len(positions), 64, torch.float32, 5)
    for interleaved in (False, True):
        got, none = K.rotary(q, None, positions, freq, interleaved=interleaved)
        assert none is None
        _check(got, q, positions, freq, interleaved, 0, 1.0)
    assert torch.equal(K.rotary(q, None, positions.int(), freq)[0], K.rotary(q, None, positions, freq)[0])
    # a frequency of a quarter of a turn, or of whole turns, at any distance: exact
    quarter = torch.tensor([math.pi / 2], dtype=torch.float64, device="cuda")
    x = torch.tensor([[[[1.0, 0.0]]]], device="cuda")
    for n, want in ((0, (1, 0)), (1, (0, 1)), (2, (-1, 0)), (3, (0, -1)), (4 * 10 ** 6 + 1, (0, 1))):
        y, _ = K.rotary(x, None, torch.tensor([n], device="cuda"), quarter)
        assert (y.flatten().cpu() - torch.tensor(want, dtype=torch.float32)).abs().max() < 2.0 ** -21 + n * 2.0 ** -50


@pytest.mark.gpu
def test_rows_of_infinities_and_nan_keep_to_themselves():
    from cinnamon_b200 import kernels as K
    q = _heads(2, 3, 9, 96, torch.bfloat16, 6)
    freq, _ = K.rotary_frequencies(32, device="cuda")
    positions = torch.arange(9, device="cuda")
    clean, _ = K.rotary(q, None, positions, freq, start=16)
    bad = q.clone()
    bad[1, 2, 4], bad[0, 0, 0] = float("nan"), float("inf")
    dirty, _ = K.rotary(bad, None, positions, freq, start=16)
    same = torch.ones(2, 3, 9, dtype=torch.bool, device="cuda")
    same[1, 2, 4] = same[0, 0, 0] = False
    assert torch.equal(dirty[same], clean[same]) and torch.isnan(dirty[1, 2, 4]).all()


@pytest.mark.gpu
def test_odd_strides_expanded_heads_and_empty():
    from cinnamon_b200 import kernels as K
    freq, _ = K.rotary_frequencies(16, device="cuda")
    base = torch.randn(2, 7, 3, 41, device="cuda").bfloat16()
    positions = torch.arange(7, device="cuda")
    for q in (base.transpose(1, 2)[..., 3:35], base.transpose(1, 2)[..., ::2], base.transpose(1, 2)[..., 1:33:1][:, :2], base.permute(0, 3, 1, 2)):
        freq_q = freq[:1] if q.shape[-1] < 16 else freq
        got, _ = K.rotary(q, None, positions, freq_q)
        _check(got, q, positions, freq_q, False, 0, 1.0)
    # one key for all heads: the expanded view, and the gradient that comes back to it
    k = torch.randn(2, 1, 7, 32, device="cuda").bfloat16().requires_grad_(True)
    g = torch.randn(2, 4, 7, 32, device="cuda").bfloat16()
    out, _ = K.rotary(k.expand(2, 4, 7, 32), None, positions, freq)
    _check(out.detach(), k.detach().expand(2, 4, 7, 32), positions, freq, False, 0, 1.0)
    dk, = torch.autograd.grad(out, k, g)
    per_head, _ = K._host.rotary(g, None, positions, freq, False, 0, 1.0, True)
    assert torch.allclose(dk.float(), per_head.float().sum(1, keepdim=True), atol=2.0 ** -5, rtol=2.0 ** -7)
    # a gradient that is itself expanded
    q = torch.randn(2, 4, 7, 32, device="cuda").requires_grad_(True)
    dq, = torch.autograd.grad(K.rotary(q, None, positions, freq)[0].sum(), q)
    _check(dq, torch.ones_like(q), positions, freq, False, 0, 1.0, inverse=True)
    # only one of the two is used
    k = torch.randn(2, 1, 7, 32, device="cuda").requires_grad_(True)
    oq, ok = K.rotary(q, k, positions, freq)
    assert torch.autograd.grad(ok.sum(), [q, k], allow_unused=True)[0] is None
    for shape in ((0, 4, 7, 32), (2, 0, 7, 32), (2, 4, 0, 32)):
        e = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        p = torch.arange(shape[2], device="cuda")
        oq, ok = K.rotary(e, torch.zeros(shape[0], 2, shape[2], 32, device="cuda", dtype=torch.bfloat16), p, freq)
        assert oq.shape == shape and ok.shape == (shape[0], 2, shape[2], 32)


@pytest.mark.gpu
def test_in_place_on_parts_of_a_fused_projection():
    """q and k as views of one (batch, L, 3, heads, d) projection; v and what is not rotated stay as they were."""
    from cinnamon_b200 import kernels as K
    qkv = torch.randn(2, 11, 3, 4, 64, device="cuda").half()
    freq, _ = K.rotary_frequencies(32, device="cuda")
    positions = torch.arange(11, device="cuda") + 5
    before = qkv.clone()
    q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    want = K.rotary(q, k, positions, freq, start=-32)
    K.rotary_(q, k, positions, freq, start=-32)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, :, 2], before[:, :, 2]) and torch.equal(qkv[..., :32], before[..., :32])


@pytest.mark.gpu
def test_streams_and_replayed_graphs():
    from cinnamon_b200 import kernels as K
    freq, _ = K.rotary_frequencies(64, device="cuda")
    q, k = _heads(4, 8, 1, 192, torch.bfloat16, 7), _heads(4, 1, 1, 576, torch.bfloat16, 8)
    positions = torch.tensor([[3], [99], [1000000], [7]], device="cuda")
    ref = K.rotary(q, k, positions, freq, start=-64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        other = K.rotary(q, k, positions, freq, start=-64)
        with torch.cuda.graph(graph, stream=side):
            captured = K.rotary(q, k, positions, freq, start=-64)
    torch.cuda.synchronize()
    assert torch.equal(other[0], ref[0]) and torch.equal(other[1], ref[1])
    positions += 17
    want = K.rotary(q, k, positions, freq, start=-64)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A last sequence that starts behind 2^31 elements."""
    from cinnamon_b200 import kernels as K
    freq, _ = K.rotary_frequencies(64, device="cuda")
    cache = torch.zeros(2, 1 << 20, 16, 72, device="cuda", dtype=torch.bfloat16)            # 2.4e9 elements
    k = cache[:, -3:].transpose(1, 2)
    k.copy_(torch.randn(2, 16, 3, 72, device="cuda"))
    positions = torch.arange(3, device="cuda") + (1 << 20) - 3
    want = K.rotary(k.contiguous(), None, positions, freq, start=8)[0]
    assert torch.equal(K.rotary(k, None, positions, freq, start=8)[0], want)
    K.rotary_(k, None, positions, freq, start=8)
    assert torch.equal(k, want) and (cache[:, :-3] == 0).all()


@pytest.mark.gpu
def test_refusals():
    from cinnamon_b200 import kernels as K
    freq, _ = K.rotary_frequencies(16, device="cuda")
    q = torch.randn(2, 3, 5, 32, device="cuda")
    k = torch.randn(2, 1, 5, 32, device="cuda")
    p = torch.arange(5, device="cuda")
    for args, what in [((q[0], k, p, freq), "batch, heads"), ((q, k.half(), p, freq), "agree"), ((q, k[:, :, :4], p, freq), "agree"),
                       ((q, k, p[:4], freq), "positions are"), ((q, k, p.float(), freq), "int64"), ((q, k, p, freq.half()), "float64"),
                       ((q.double(), None, p, freq), "bfloat16"), ((q, k, p.cpu(), freq), "CUDA"), ((q, k, p, freq.repeat(3)), "do not fit")]:
        with pytest.raises(AssertionError, match=what):
            K.rotary(*args)
    with pytest.raises(AssertionError, match="no gradient"):
        K.rotary(q, k, p, freq.clone().requires_grad_(True))
    for start in (17, -15, -33):
        with pytest.raises(AssertionError, match="do not fit"):
            K.rotary(q, k, p, freq, start=start)
    with pytest.raises(AssertionError, match="expanded"):
        K.rotary_(k.expand(2, 3, 5, 32), None, p, freq)
    with pytest.raises(AssertionError, match="same memory"):
        K.rotary_(q, q, p, freq)
    with pytest.raises(AssertionError, match="differentiable"):
        K.rotary_(q.clone().requires_grad_(True), None, p, freq)
    a = q.clone().requires_grad_(True)
    with pytest.raises(AssertionError, match="second derivative"):
        torch.autograd.grad(K.rotary(a, None, p, freq)[0].sum(), a, create_graph=True)


def test_frequencies():
    from cinnamon_b200 import kernels as K
    f, m = K.rotary_frequencies(8, base=10000.0)
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(K.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4)
    ntk, _ = K.rotary_frequencies(8, scaling="ntk", factor=16.0)
    assert ntk[0] == 1.0 and abs(float(ntk[-1] * 16 / f[-1]) - 1) < 1e-12
    y, m = K.rotary_frequencies(64, scaling="yarn", factor=32.0, original_len=4096, mscale=0.5)
    g, _ = K.rotary_frequencies(64)
    assert abs(m - (0.05 * math.log(32.0) + 1)) < 1e-15
    assert torch.equal(y[0], g[0]) and torch.allclose(y[-1], g[-1] / 32, rtol=1e-14)
    assert ((y <= g) & (y >= g / 32 * (1 - 1e-14))).all()
    turns = g * 4096 / (2 * math.pi)
    assert torch.equal(y[turns > 45], g[turns > 45])
    for bad in (dict(dim=7), dict(dim=8, scaling="other"), dict(dim=8, scaling="yarn", factor=2.0), dict(dim=8, factor=0.5)):
        with pytest.raises(AssertionError):
            K.rotary_frequencies(**bad)


def test_a_cpu_tensor_is_refused():
    from cinnamon_b200 import kernels as K
    q = torch.randn(1, 2, 3, 16)
    with pytest.raises(AssertionError, match="CUDA"):
        K.rotary(q, None, torch.arange(3), K.rotary_frequencies(16)[0])
