"""What stands around the framework's layers in a language model's step, as timed cases over the public entry points.

  loss_train     ``linear_cross_entropy``: the output projection and its cross entropy, loss and both gradients
  loss_eval      the same without gradients, one loss per token: evaluation, scoring of answers
  rotary_train   ``rotary`` on queries and keys as sparse attention takes them, and the gradients through it
  rotary_serve   ``rotary`` without gradients: prefill and decoding, positions far into a long context
  route_train    ``moe_route`` on softmax scores or groups of experts, and the gradient of the gates
  route_serve    ``moe_route`` without gradients: groups of experts, a bias for balance, scaled gates

Sizes are those of the repository's benchmark (a 512-wide model of 32000 tokens' vocabulary trained on 32 x 1024 tokens,
7168-wide layers, attention of 128 heads of 192 of which 64 are rotated, 256 experts on 32768 tokens) or generic ones;
``draw`` spreads over the ranges between them.  The plain form writes the formulas in elementary torch operations.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ITEM = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORED = -100


def listed():
    return [
        # the head of the narrow model in training: 32 x 1024 tokens, every one of them a target
        dict(name="loss_train_narrow", kind="loss_train", tokens=32768, valid=32768, d=512, vocab=32000, dtype="bf16"),
        # the head of a wide model on one long sequence, a large vocabulary
        dict(name="loss_train_wide", kind="loss_train", tokens=4096, valid=4096, d=7168, vocab=128000, dtype="bf16"),
        # fine-tuning on answers: the prompts and the padding are ignored, nothing is a multiple of a tile
        dict(name="loss_train_answers", kind="loss_train", tokens=8191, valid=3001, d=2040, vocab=50003, dtype="fp16"),
        # a short sequence on one GPU: the weight's gradient is nearly all the memory there is to move
        dict(name="loss_train_short", kind="loss_train", tokens=130, valid=130, d=512, vocab=32000, dtype="bf16"),
        # scoring one prompt of an odd length, a loss for each token
        dict(name="loss_eval_prompt", kind="loss_eval", tokens=1531, valid=1531, d=512, vocab=32000, dtype="bf16"),
        # queries and keys of the narrow model's sparse attention in training: the last 64 of 192 are rotated
        dict(name="rotary_train", kind="rotary_train", batch=32, seq=1024, heads=8, kv_heads=8, d=192, d_kv=192, rot=64, interleaved=False,
             scaling="none", seq_first=False, first=0, dtype="bf16"),
        # prefill of wide attention: 128 heads as the projection leaves them, one shared key of 512 + 64, far into a long context
        dict(name="rotary_prefill", kind="rotary_serve", batch=4, seq=4096, heads=128, kv_heads=1, d=192, d_kv=576, rot=64, interleaved=True,
             scaling="yarn", seq_first=True, first=100000, dtype="bf16"),
        # decoding for 64 sequences, each at a position of its own: launches and host work
        dict(name="rotary_decode", kind="rotary_serve", batch=64, seq=1, heads=128, kv_heads=1, d=192, d_kv=576, rot=64, interleaved=True,
             scaling="yarn", seq_first=True, first=-1, dtype="bf16"),
        # the wide layer's router on a prefill batch: 8 of 256 experts out of 4 of 8 groups
        dict(name="route_prefill", kind="route_serve", tokens=32768, experts=256, top_k=8, scores="sigmoid", groups=8, top_groups=4,
             renormalise=True, scale=2.5, bias_std=0.1, dtype="bf16"),
        # the same router generating for 64 sequences
        dict(name="route_decode", kind="route_serve", tokens=64, experts=256, top_k=8, scores="sigmoid", groups=8, top_groups=4,
             renormalise=True, scale=2.5, bias_std=0.1, dtype="bf16"),
        # a softmax router in training, gates as they come out of the softmax
        dict(name="route_train", kind="route_train", tokens=16384, experts=64, top_k=6, scores="softmax", groups=1, top_groups=1,
             renormalise=False, scale=1.0, bias_std=0.0, dtype="fp32"),
        # the narrow model's 16 experts in training, on softmax scores
        dict(name="route_train_narrow", kind="route_train", tokens=32768, experts=16, top_k=2, scores="softmax", groups=1, top_groups=1,
             renormalise=True, scale=1.0, bias_std=0.0, dtype="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return min(max(v, lo), hi)


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 6.0 * 4096 * 128000 * 7168 and w["bytes"] <= 6e9:
            return case


def _draw(rng):
    kind = rng.choice(["loss_train", "loss_train", "loss_eval", "rotary_train", "rotary_serve", "rotary_serve", "route_train", "route_serve"])
    if kind.startswith("loss"):
        tokens = _log(rng, 1, 32768)
        valid = tokens if rng.random() < 0.5 else max(1, int(tokens * rng.uniform(0.1, 1.0)))
        # the plain form holds tokens x vocabulary in 32 bits a few times over
        vocab = _log(rng, 1000, min(160000, int(1.1e9) // tokens))
        return dict(kind=kind, tokens=tokens, valid=valid, d=_log(rng, 64, 7168, 8), vocab=vocab, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind.startswith("rotary"):
        heads = rng.choice([1, 8, 16, 32, 128])
        d = rng.choice([64, 96, 128, 192])
        return dict(kind=kind, batch=_log(rng, 1, 64), seq=_log(rng, 1, 16384), heads=heads, kv_heads=rng.choice([h for h in (1, 2, 8, 32) if h <= heads]),
                    d=d, d_kv=rng.choice([d, d, 576]), rot=rng.choice([r for r in (32, 64, 128) if r <= d]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn"]), seq_first=rng.random() < 0.5,
                    first=rng.choice([-1, 0, 0, _log(rng, 1, 1000000)]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    experts = rng.choice([8, 16, 60, 64, 128, 160, 256])
    scores = rng.choice(["sigmoid", "softmax"])
    groups = rng.choice([g for g in (1, 4, 8) if experts % g == 0 and experts // g >= 2]) if scores == "softmax" else rng.choice([2, 4])
    top_groups = rng.randint(1, groups)
    return dict(kind=kind, tokens=_log(rng, 1, 65536), experts=experts, top_k=rng.randint(1, min(8, top_groups * (experts // groups))), scores=scores,
                groups=groups, top_groups=top_groups, renormalise=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                bias_std=rng.choice([0.0, 0.1]), dtype=rng.choice(["bf16", "fp32", "fp16"]))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _inv_freq(c, device):
    """Frequencies in radians a position, in 64 bits, and the factor on the rotated values."""
    base, factor, original = 10000.0, 32.0, 4096
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device=device)
    freq = base ** (-2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        return freq / factor, 1.0
    if c["scaling"] == "yarn":
        turns = lambda r: c["rot"] * math.log(original / (2 * math.pi * r)) / (2 * math.log(base))      # noqa: E731
        low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), c["rot"] - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)                                         # noqa: E731
    dt = DTYPES[c["dtype"]]
    s = dict(case=c, kind=kind)
    if kind.startswith("loss"):
        T, V, d = c["tokens"], c["vocab"], c["d"]
        w = (randn(V, d) * 0.02).to(dt)
        target = torch.randint(0, V, (T,), generator=g, device=DEV)
        # tokens of a model under training: some predicted well, most not
        lift = torch.rand(T, generator=g, device=DEV).pow(3) * 12.0
        hit = w[target].float()
        x = (randn(T, d) + lift[:, None] * hit / hit.pow(2).sum(-1, keepdim=True)).to(dt)
        if c["valid"] < T:
            target[torch.randperm(T, generator=g, device=DEV)[:T - c["valid"]]] = IGNORED
        s.update(x=x, w=w, target=target)
        if kind == "loss_train":
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
            # 16-bit floats of a short exponent are trained with a scaled loss
            s["d_loss"] = torch.tensor(4096.0 if c["dtype"] == "fp16" else 1.0, device=DEV)
        return s
    if kind.startswith("rotary"):
        B, L = c["batch"], c["seq"]

        def heads(h, d):                              # (batch, heads, positions, d), stored so or positions first
            return randn(B, L, h, d).to(dt).transpose(1, 2) if c["seq_first"] else randn(B, h, L, d).to(dt)

        s.update(q=heads(c["heads"], c["d"]), k=heads(c["kv_heads"], c["d_kv"]))
        if c["first"] < 0:                            # every sequence somewhere else
            first = torch.randint(0, 1000000, (B, 1), generator=g, device=DEV)
            s["positions"] = first + torch.arange(L, device=DEV)
        else:
            s["positions"] = torch.arange(c["first"], c["first"] + L, device=DEV)
        s["inv_freq"], s["magnitude"] = _inv_freq(c, DEV)
        if kind == "rotary_train":
            s["dq"], s["dk"] = heads(c["heads"], c["d"]), heads(c["kv_heads"], c["d_kv"])
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
        return s
    T, E = c["tokens"], c["experts"]
    s["logits"] = (randn(T, E) * 1.5).to(dt)
    s["bias"] = randn(E) * c["bias_std"]
    if kind == "route_train":
        s["logits"].requires_grad_(True)
        s["d_gates"] = randn(T, c["top_k"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        if s["kind"].startswith("loss"):
            return _loss_plain(s)
        if s["kind"].startswith("rotary"):
            return _rotary_plain(s)
        return _route_plain(s)


def _run_own(s):
    from cinnamon_b200 import kernels as K
    kind, c = s["kind"], s["case"]
    if kind == "loss_train":
        loss = K.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORED)
        gx, gw = torch.autograd.grad(loss, [s["x"], s["w"]], s["d_loss"])
        return dict(loss=loss.detach(), grad_x=gx, grad_w=gw)
    if kind == "loss_eval":
        with torch.no_grad():
            return K.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORED, reduction="none")
    if kind.startswith("rotary"):
        form = dict(interleaved=c["interleaved"], start=-c["rot"], magnitude=s["magnitude"])
        q, k = K.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], **form)
        if kind == "rotary_serve":
            return dict(q=q, k=k)
        gq, gk = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])
        return dict(q=q.detach(), k=k.detach(), grad_q=gq, grad_k=gk)
    r = K.moe_route(s["logits"], s["bias"], c["top_k"], scores=c["scores"], n_groups=c["groups"], top_groups=c["top_groups"],
                    renormalise=c["renormalise"], scale=c["scale"])
    out = {name: r[name].detach() for name in ("top_experts", "top_gates", "token_indices", "sorted_scores", "sorted_experts", "counts", "starts",
                                               "ends", "pair_pos", "pair_gate")}
    if kind == "route_train":
        out["grad_logits"], = torch.autograd.grad(r["top_gates"], s["logits"], s["d_gates"])
    return out


def _loss_plain(s):
    x, w, target = s["x"].float(), s["w"].float(), s["target"]
    keep = target != IGNORED
    safe = target.clamp(min=0)[:, None]
    z = x @ w.t()
    m = z.amax(-1, keepdim=True)
    e = (z - m).exp()
    total = e.sum(-1, keepdim=True)
    loss = (m - z.gather(-1, safe) + total.log())[:, 0] * keep
    if s["kind"] == "loss_eval":
        return loss
    n = keep.sum()
    g = e / total
    g.scatter_add_(-1, safe, torch.full_like(m, -1.0))
    g *= keep[:, None] * (s["d_loss"] / n)
    return dict(loss=loss.sum() / n, grad_x=(g @ w).to(s["x"].dtype), grad_w=(g.t() @ x).to(s["w"].dtype))


def _rotate_plain(t, positions, inv_freq, magnitude, interleaved, sign):
    rot = 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq
    angle = angle[None, None] if angle.dim() == 2 else angle[:, None]                 # (1 or batch, 1, positions, rot / 2)
    cos, sin = (angle.cos() * magnitude).float(), (sign * angle.sin() * magnitude).float()
    rest, part = t[..., :t.shape[-1] - rot], t[..., t.shape[-1] - rot:].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([rest, turned.to(t.dtype)], -1)


def _rotary_plain(s):
    form = (s["positions"], s["inv_freq"], s["magnitude"], s["case"]["interleaved"])
    out = dict(q=_rotate_plain(s["q"], *form, 1.0), k=_rotate_plain(s["k"], *form, 1.0))
    if s["kind"] == "rotary_train":
        out.update(grad_q=_rotate_plain(s["dq"], *form, -1.0), grad_k=_rotate_plain(s["dk"], *form, -1.0))
    return out


def _scores(logits, scores):
    if scores == "sigmoid":
        return 1.0 / (1.0 + (-logits).exp())
    e = (logits - logits.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _choose_plain(s):
    """The experts of every token, by falling score + bias, ties to the lower one.  In 64 bits: scores next to one another
    decide which expert is the last."""
    c = s["case"]
    T, E, G = c["tokens"], c["experts"], c["groups"]
    chosen_by = _scores(s["logits"].double(), c["scores"]) + s["bias"].double()
    if G > 1:
        best = chosen_by.view(T, G, E // G).sort(dim=-1, descending=True).values[..., :2].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True).indices
        closed = torch.ones_like(best, dtype=torch.bool).scatter_(-1, order[:, :c["top_groups"]], False)
        chosen_by = chosen_by.masked_fill(closed.repeat_interleave(E // G, -1), -math.inf)
    return chosen_by.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_k"]]


def _route_plain(s):
    c = s["case"]
    T, E, k = c["tokens"], c["experts"], c["top_k"]
    top = _choose_plain(s)
    score = _scores(s["logits"].float(), c["scores"])
    picked = score.gather(-1, top)
    total = picked.sum(-1, keepdim=True) + 1e-9
    gates = (picked / total if c["renormalise"] else picked) * c["scale"]
    expert = top.reshape(-1)
    sorted_experts, order = expert.sort(stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(T * k, device=order.device)
    pair_pos, perm = pos.view(T, k).sort(-1)
    counts = torch.bincount(expert, minlength=E)
    ends = counts.cumsum(0)
    out = dict(top_experts=top.int(), top_gates=gates, token_indices=order // k, sorted_scores=gates.reshape(-1)[order],
               sorted_experts=sorted_experts, counts=counts, starts=ends - counts, ends=ends, pair_pos=pair_pos,
               pair_gate=gates.gather(-1, perm))
    if s["kind"] == "route_train":
        dg = s["d_gates"] * c["scale"]
        d_picked = (dg - (dg * picked).sum(-1, keepdim=True) / total) / total if c["renormalise"] else dg
        d_score = torch.zeros_like(score).scatter_(-1, top, d_picked)
        if c["scores"] == "sigmoid":
            d = d_score * score * (1 - score)
        else:
            d = score * (d_score - (d_score * score).sum(-1, keepdim=True))
        out["grad_logits"] = d.to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    c, kind = case, case["kind"]
    it = ITEM[c["dtype"]]
    if kind.startswith("loss"):
        T, n, V, d = c["tokens"], c["valid"], c["vocab"], c["d"]
        once = it * (n * d + V * d)
        if kind == "loss_eval":
            return dict(bytes=once + 12 * T, flops=2.0 * n * V * d)
        return dict(bytes=once + it * (T * d + V * d) + 8 * T + 4, flops=6.0 * n * V * d)
    if kind.startswith("rotary"):
        each = c["batch"] * c["seq"] * (c["heads"] * c["d"] + c["kv_heads"] * c["d_kv"])
        turned = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"]) * c["rot"]
        passes = 2 if kind == "rotary_train" else 1
        return dict(bytes=passes * 2 * each * it + 8 * c["seq"], flops=passes * 3.0 * turned)
    T, E, k = c["tokens"], c["experts"], c["top_k"]
    outputs = T * k * (4 + 4 + 8 + 4 + 8 + 8 + 4) + 24 * E
    if kind == "route_serve":
        return dict(bytes=it * T * E + 4 * E + outputs, flops=8.0 * T * E)
    return dict(bytes=2 * it * T * E + 4 * E + outputs + 4 * T * k, flops=16.0 * T * E)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if s["kind"].startswith("loss"):
            return _loss_exact(s)
        if s["kind"].startswith("rotary"):
            return _rotary_exact(s)
        return _route_exact(s)


def _loss_exact(s):
    """Rows in pieces: log-sum-exp, and the softmax less the target's unit vector against weight and activations."""
    x, w, target = s["x"].detach().double(), s["w"].detach().double(), s["target"]
    T, d = x.shape
    rows = torch.nonzero(target != IGNORED)[:, 0]
    losses = x.new_zeros(T)
    gx, gw = x.new_zeros(T, d), None
    step = max(1, (1 << 28) // w.shape[0])
    for at in range(0, rows.numel(), step):
        r = rows[at:at + step]
        z = x[r] @ w.T
        lse = torch.logsumexp(z, -1)
        mine = torch.arange(r.numel(), device=r.device)
        losses[r] = lse - z[mine, target[r]]
        if s["kind"] == "loss_train":
            z = torch.exp(z - lse[:, None])
            z[mine, target[r]] -= 1.0
            z *= float(s["d_loss"]) / rows.numel()
            gx[r] = z @ w
            part = z.T @ x[r]
            gw = part if gw is None else gw.add_(part)
    if s["kind"] == "loss_eval":
        return losses
    return dict(loss=losses.sum() / rows.numel(), grad_x=gx, grad_w=gw)


def _rotary_exact(s):
    """Pairs as complex numbers, turned by the unit number of their angle."""
    c = s["case"]
    at = s["positions"].double()
    angle = torch.einsum("...l,f->...lf", at, s["inv_freq"])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)
    turn = turn.unsqueeze(-3)

    def turned(t, by):
        t = t.detach().double()
        keep = t.shape[-1] - c["rot"]
        p = t[..., keep:]
        p = p.unflatten(-1, (c["rot"] // 2, 2)) if c["interleaved"] else p.unflatten(-1, (2, c["rot"] // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(p.contiguous()) * by)
        y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat([t[..., :keep], y], -1)

    out = dict(q=turned(s["q"], turn), k=turned(s["k"], turn))
    if s["kind"] == "rotary_train":
        out.update(grad_q=turned(s["dq"], turn.conj()), grad_k=turned(s["dk"], turn.conj()))
    return out


def _route_exact(s):
    """Expert by expert: rounds of "the best one left", gates and their derivative through autograd in 64 bits."""
    c = s["case"]
    T, E, G, k = c["tokens"], c["experts"], c["groups"], c["top_k"]
    logits = s["logits"].detach().double().requires_grad_(True)
    with torch.enable_grad():
        score = torch.sigmoid(logits) if c["scores"] == "sigmoid" else torch.softmax(logits, -1)
        left = (score + s["bias"].double()).detach().clone()
        rows = torch.arange(T, device=logits.device)
        if G > 1:
            per = left.view(T, G, E // G)
            first = per.max(-1)
            rest = per.clone()
            rest[rows[:, None], torch.arange(G, device=rows.device)[None], first.indices] = -math.inf
            groups = first.values + rest.max(-1).values
            is_open = torch.zeros(T, G, dtype=torch.bool, device=rows.device)
            for _ in range(c["top_groups"]):
                best = (groups == groups.max(-1, keepdim=True).values).int().argmax(-1)        # the first of the largest
                is_open[rows, best] = True
                groups[rows, best] = -math.inf
            left[~is_open.repeat_interleave(E // G, dim=1)] = -math.inf
        top = torch.empty(T, k, dtype=torch.int64, device=rows.device)
        for j in range(k):
            top[:, j] = (left == left.max(-1, keepdim=True).values).int().argmax(-1)
            left[rows, top[:, j]] = -math.inf
        gates = torch.take_along_dim(score, top, 1)
        if c["renormalise"]:
            gates = gates / (gates.sum(1, keepdim=True) + 1e-9)
        gates = gates * c["scale"]
    flat, g = top.reshape(-1), gates.detach()
    # the place of every pair: all pairs of lower experts, and the earlier pairs of its own
    order = torch.argsort(flat * (T * k) + torch.arange(T * k, device=flat.device))
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=flat.device)
    place = place.view(T, k)
    by_place = torch.argsort(place, dim=1)
    counts = torch.zeros(E, dtype=torch.int64, device=flat.device).index_add_(0, flat, torch.ones_like(flat))
    ends = torch.cumsum(counts, 0)
    out = dict(top_experts=top.int(), top_gates=g, token_indices=torch.div(order, k, rounding_mode="floor"), sorted_scores=g.reshape(-1)[order],
               sorted_experts=flat[order], counts=counts, starts=ends - counts, ends=ends, pair_pos=torch.take_along_dim(place, by_place, 1),
               pair_gate=torch.take_along_dim(g, by_place, 1))
    if s["kind"] == "route_train":
        out["grad_logits"], = torch.autograd.grad(gates, logits, s["d_gates"].double())
    return out
