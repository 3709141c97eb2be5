"""What ``linear_cross_entropy``'s operators look at before anything reaches a kernel; no GPU is needed for it (tensors without memory stand for those of one)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def _operands(T=6, V=20, d=64):
    x, w = torch.empty(T, d, dtype=torch.bfloat16, device="cuda"), torch.empty(V, d, dtype=torch.bfloat16, device="cuda")
    return x, w, torch.empty(T, dtype=torch.int64, device="cuda")


def test_operators_of_a_compiled_graph_refuse_what_the_kernels_cannot_read():
    from cinnamon_b200 import kernels as K
    forward, backward, finish = K._host.linear_ce_forward, K._host.linear_ce_backward, K._host.linear_ce_finish
    with FakeTensorMode():
        x, w, t = _operands()
        here = dict(dtype=torch.bfloat16)
        for a, b, c, what in [(torch.empty(6, 64, **here), torch.empty(20, 64, **here), torch.empty(6, dtype=torch.int64), "CUDA"),
                              (x, torch.empty(20, 64, **here), t, "CUDA"), (x, w, torch.empty(6, dtype=torch.int64), "same device"),
                              (x, w, t[:5], "one int64"), (x, w, t.int(), "one int64"), (x, w, t[:, None], "one int64"), (x, w[:, :56], t, "multiple of 8"),
                              (x[:, :60], w[:, :60], t, "multiple of 8"), (x, w[:0], t, "multiple of 8"), (x[None], w, t, "multiple of 8"),
                              (x, w.half(), t, "16-bit"), (x.float(), w.float(), t, "16-bit")]:
            with pytest.raises(AssertionError, match=what):
                forward(a, b, c, -100, 1, False)
        one, each = torch.empty((), device="cuda"), torch.empty(6, device="cuda")
        state = torch.empty(256 * 6, dtype=torch.uint8, device="cuda")
        none = torch.empty(0, device="cuda")
        for grad, reduction, kept, what in [(one.cpu(), 1, state, "gradient"), (each, 1, state, "gradient"), (one, 0, state, "gradient"),
                                            (one, 1, state[:5], "left for"), (one, 1, state.cpu(), "left for"), (one, 1, state.float(), "left for")]:
            with pytest.raises(AssertionError, match=what):
                backward(grad, x, w, kept, reduction, True, True)
        for grad, reduction, kept, what in [(one.cpu(), 1, state, "gradient"), (each, 1, state, "gradient"), (one, 0, state, "sum or mean"),
                                            (one, 1, state[:5], "left for"), (one, 1, state.cpu(), "CUDA"), (one, 1, state.float(), "left for")]:
            with pytest.raises(AssertionError, match=what):
                finish(grad, kept, none, none, 6, 20, 64, torch.bfloat16, reduction, True, True)
        for shape in ((0, 20, 64), (6, 0, 64), (6, 20, 63)):
            with pytest.raises(AssertionError, match="sum or mean"):
                finish(one, state, none, none, *shape, torch.bfloat16, 1, True, True)
        with pytest.raises(AssertionError, match="sum or mean"):
            finish(one, state, none, none, 6, 20, 64, torch.float32, 1, True, True)


def test_workspaces_are_what_the_documentation_says():
    """Sizes alone decide on them: a copy of x's rows, the parts of the statistics, a piece of the logits' gradient, x's gradient in fp32 (and
    where a product's sums are cut for want of tiles, at most one 256 x 256 tile of sums for each pair of SMs)."""
    from cinnamon_b200._lib import lib as L
    MiB = 1 << 20
    for T in (1, 100, 2048, 4096, 8191, 32768, 65537, 1 << 20, 3 << 20):
        for V in (1, 300, 32000, 128000, 262144, 1 << 20):
            for d in (8, 512, 1024, 2040, 7168, 16384):
                if T * d > 1 << 33:
                    continue
                Tp, rows = (T + 255) // 256 * 256, 2 * T * d
                piece, small = max(512 * MiB, 512 * Tp), 70 * MiB + 40 * T
                tiles = 4 * 256 * 256 * 80
                assert L.cinn_linear_ce_workspace_bytes(T, V, d, 0) <= rows + small, (T, V, d)
                assert L.cinn_linear_ce_workspace_bytes(T, V, d, 1) <= rows + small + max(1300 * MiB, 520 * V), (T, V, d)
                assert L.cinn_linear_ce_workspace_bytes(T, V, d, 5) <= rows + piece + max(4 * Tp * d, tiles) + small, (T, V, d)
                assert L.cinn_linear_ce_workspace_bytes(T, V, d, 6) <= rows + piece + tiles + small, (T, V, d)
                assert L.cinn_linear_ce_workspace_bytes(T, V, d, 7) <= rows + piece + max(4 * Tp * d, tiles) + tiles + small, (T, V, d)
                assert L.cinn_linear_ce_state_bytes(T) <= 20 * T + 5 * 256
                if L.cinn_linear_ce_early(T, V, d, 1, 0):
                    sums = [L.cinn_linear_ce_early(T, V, d, 1, i) for i in (1, 2)]
                    pieces = -(-Tp // max(256, (1280 * MiB // (2 * (V + 63))) // 256 * 256))
                    assert sum(sums) <= 8 << 30 and sums[0] <= max(4 * Tp * d, pieces * tiles) and sums[1] <= max(4 * (V + 255) * d, tiles), (T, V, d)
