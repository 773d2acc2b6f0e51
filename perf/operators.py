"""What the operators around a block of routed experts are measured on: the norm in front of it, the choice of the experts, and the
experts themselves for a few tokens.

* ``experts``  a whole layer of routed SwiGLU experts for 1 to 32 tokens (a decode step), weights in bf16 or in e4m3 with one fp32 scale
               per block of 128 x 128; optionally only the experts that this rank holds;
* ``norm``     the residual's addition and the root-mean-square norm, for serving with the rows of the FP8 dispatch beside the bf16 rows,
               for training with its gradients;
* ``route``    the k largest of a token's gate logits and their weights, for training with the logits' gradient.

Sizes are those of the benchmarks' layers (hidden 7168, 256 experts of 7168 -> 2048, top-8; hidden 4096, 64 experts of 4096 -> 1408, top-6;
4096 and 8192 tokens; one token up to 32 in a decode step), smaller and ragged ones of the same kind, and in ``draw`` what lies between.
``run`` computes each operator in elementary torch operations in 32 bits, or with ``own`` through the framework's entry points.
"""
import math

import torch

own = False
DEVICE = "cuda"
EPS = 1e-6


def listed():
    return [
        # one token through a small layer: nothing but latency, ragged widths, a selection that was dropped
        dict(name="experts_3_small", kind="experts", tokens=3, hidden=1032, inter=648, experts=16, local=16, topk=2, fp8=False, dropped=0.2),
        # one user's decode step, bf16 weights
        dict(name="experts_1_bf16", kind="experts", tokens=1, hidden=4096, inter=1408, experts=64, local=64, topk=6, fp8=False, dropped=0.0),
        # the same step of the large layer in FP8
        dict(name="experts_1_fp8", kind="experts", tokens=1, hidden=7168, inter=2048, experts=256, local=256, topk=8, fp8=True, dropped=0.0),
        # eight users of the large layer
        dict(name="experts_8_fp8", kind="experts", tokens=8, hidden=7168, inter=2048, experts=256, local=256, topk=8, fp8=True, dropped=0.0),
        # a ragged batch of the smaller layer: most experts are read, by a token or two each
        dict(name="experts_20_bf16", kind="experts", tokens=20, hidden=4096, inter=1408, experts=64, local=64, topk=6, fp8=False, dropped=0.0),
        # the largest batch, on one of four ranks that share the large layer's experts
        dict(name="experts_32_fp8_share", kind="experts", tokens=32, hidden=7168, inter=2048, experts=256, local=64, topk=8, fp8=True, dropped=0.0),
        # decode: one row, its sum with the residual, and both forms of the normed row
        dict(name="norm_1_fp8", kind="norm", tokens=1, hidden=7168, residual=True, fp8=True, train=False, wide=False),
        # the benchmark's prefill batch in front of an FP8 dispatch
        dict(name="norm_4096_fp8", kind="norm", tokens=4096, hidden=7168, residual=True, fp8=True, train=False, wide=False),
        # the benchmark's training batch, forward and backward
        dict(name="norm_train_8192", kind="norm", tokens=8192, hidden=4096, residual=True, fp8=False, train=True, wide=True),
        # one token's choice
        dict(name="route_1", kind="route", tokens=1, experts=256, topk=8, renormalize=True, train=False, bf16=False, masked=0.0),
        # the training batch of the smaller layer with its gradient
        dict(name="route_train_8192", kind="route", tokens=8192, experts=64, topk=6, renormalize=True, train=True, bf16=False, masked=0.0),
        # a ragged batch of bf16 logits (ties), some experts taken out, probabilities among all experts
        dict(name="route_train_3001", kind="route", tokens=3001, experts=256, topk=8, renormalize=False, train=True, bf16=True, masked=0.1),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """Any kind: 1 to 32 tokens through 8 to 256 experts of hidden 1024 to 7168; norms of 1 to 8192 rows; choices of 1 to 8192 tokens among 8 to 256."""
    kind = rng.choice(("experts", "experts", "norm", "route"))
    if kind == "experts":
        fp8 = rng.random() < 0.5
        experts = rng.choice((8, 16, 32, 64, 128, 256) if fp8 else (8, 16, 32, 64))
        local = experts if rng.random() < 0.7 else experts // 2
        tokens, topk = _log_int(rng, 1, 32), rng.randint(1, 8)
        if fp8:
            hidden, inter = 128 * rng.randint(8, 56), 128 * rng.randint(4, 16)
        else:
            hidden, inter = 8 * rng.randint(128, 512), 8 * rng.randint(64, 176)
        return dict(kind=kind, tokens=tokens, hidden=hidden, inter=inter, experts=experts, local=local, topk=topk, fp8=fp8, dropped=rng.choice((0.0, 0.0, 0.15)))
    if kind == "norm":
        train = rng.random() < 0.5
        hidden = 128 * rng.randint(8, 56) if not train else 8 * rng.randint(128, 896)
        return dict(kind=kind, tokens=_log_int(rng, 1, 8192 * 4096 // max(4096, hidden)), hidden=hidden, residual=rng.random() < 0.7, fp8=not train, train=train,
                    wide=rng.random() < 0.5)
    return dict(kind=kind, tokens=_log_int(rng, 1, 8192), experts=rng.choice((8, 16, 60, 64, 128, 160, 256)), topk=rng.randint(1, 8), renormalize=rng.random() < 0.5,
                train=rng.random() < 0.7, bf16=rng.random() < 0.5, masked=rng.choice((0.0, 0.1)))


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _weights(n, rows, cols, fp8, g):
    """``n`` experts' matrices as a trained layer has them (normal, 0.02), quantised per block of 128 x 128 where ``fp8``."""
    if not fp8:
        w = torch.empty(n, rows, cols, dtype=torch.bfloat16, device=DEVICE)
        for e in range(n):
            w[e].normal_(0.0, 0.02, generator=g)
        return w, None
    w = torch.empty(n, rows, cols, dtype=torch.float8_e4m3fn, device=DEVICE)
    s = torch.empty(n, rows // 128, cols // 128, dtype=torch.float32, device=DEVICE)
    for e in range(n):
        b = torch.empty(rows // 128, 128, cols // 128, 128, dtype=torch.float32, device=DEVICE).normal_(0.0, 0.02, generator=g)
        s[e] = b.abs().amax(dim=(1, 3)) / 448.0
        w[e] = (b / s[e][:, None, :, None]).view(rows, cols).to(torch.float8_e4m3fn)
    return w, s


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    c, T = case, case["tokens"]

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype)

    if c["kind"] == "experts":
        w13, s13 = _weights(c["local"], 2 * c["inter"], c["hidden"], c["fp8"], g)
        w2, s2 = _weights(c["local"], c["hidden"], c["inter"], c["fp8"], g)
        idx = torch.rand(T, c["experts"], generator=g, device=DEVICE).topk(c["topk"], dim=-1).indices
        weights = torch.softmax(normal(T, c["topk"], dtype=torch.float32), dim=-1)
        idx = torch.where(torch.rand(T, c["topk"], generator=g, device=DEVICE) < c["dropped"], torch.full_like(idx, -1), idx)
        return dict(kind="experts", x=normal(T, c["hidden"]), idx=idx, weights=weights, w13=w13, s13=s13, w2=w2, s2=s2, first=c["experts"] - c["local"])
    if c["kind"] == "norm":
        H = c["hidden"]
        return dict(kind="norm", x=normal(T, H), residual=normal(T, H, std=3.0) if c["residual"] else None,
                    weight=(1.0 + 0.2 * torch.randn(H, generator=g, device=DEVICE)).to(torch.float32 if c["wide"] else torch.bfloat16),
                    train=c["train"], dy=normal(T, H, std=0.1) if c["train"] else None, ds=normal(T, H, std=0.1) if c["train"] and c["residual"] else None)
    logits = normal(T, c["experts"], dtype=torch.bfloat16 if c["bf16"] else torch.float32, std=1.5)
    if c["masked"]:
        logits[:, torch.rand(c["experts"], generator=g, device=DEVICE) < c["masked"]] = -math.inf
    return dict(kind="route", logits=logits, topk=c["topk"], renormalize=c["renormalize"], dw=normal(T, c["topk"], dtype=torch.float32) if c["train"] else None)


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"experts": _plain_experts, "norm": _plain_norm, "route": _plain_route}[state["kind"]](state)


def _own(s):
    if s["kind"] == "experts":
        from deepep_efa_b200.ops.few_tokens import few_token_experts
        return few_token_experts(s["x"], s["idx"], s["weights"], s["w13"], s["w2"], w13_scales=s["s13"], w2_scales=s["s2"], first_expert=s["first"])
    if s["kind"] == "norm":
        from deepep_efa_b200.ops.norm import rms_norm, rms_norm_fp8
        if not s["train"]:
            (q, scales), y, total = rms_norm_fp8(s["x"], s["weight"], s["residual"], eps=EPS)
            return dict(q=q, scales=scales, y=y, total=total)
        x, weight = s["x"].detach().requires_grad_(True), s["weight"].detach().requires_grad_(True)
        if s["residual"] is None:
            y = rms_norm(x, weight, eps=EPS)
            gx, gw = torch.autograd.grad(y, (x, weight), s["dy"])
            return dict(y=y.detach(), total=None, gx=gx, gr=None, gw=gw)
        residual = s["residual"].detach().requires_grad_(True)
        y, total = rms_norm(x, weight, residual, eps=EPS)
        gx, gr, gw = torch.autograd.grad((y, total), (x, residual, weight), (s["dy"], s["ds"]))
        return dict(y=y.detach(), total=total.detach(), gx=gx, gr=gr, gw=gw)
    from deepep_efa_b200.ops.router import select_experts
    if s["dw"] is None:
        idx, weights = select_experts(s["logits"], s["topk"], renormalize=s["renormalize"])
        return dict(idx=idx, weights=weights, dlogits=None)
    logits = s["logits"].detach().requires_grad_(True)
    idx, weights = select_experts(logits, s["topk"], renormalize=s["renormalize"])
    (dlogits,) = torch.autograd.grad(weights, logits, s["dw"])
    return dict(idx=idx, weights=weights.detach(), dlogits=dlogits)


def _plain_experts(s):
    """y[t] = sum_k weights[t, k] * W2[e] (silu(G[e] x[t]) * (U[e] x[t])) with e = idx[t, k], over the experts that are here; those that no token chose are not read."""
    local = s["idx"] - s["first"]
    here = (local >= 0) & (local < s["w13"].size(0)) & (s["idx"] >= 0)
    experts = torch.unique(local[here])
    share = ((local[None] == experts[:, None, None]) & here[None]) * s["weights"][None]  # [active, T, K]

    def wide(w, scales):
        w = w[experts].float() if scales is None else w.view(torch.uint8)[experts].view(w.dtype).float()
        if scales is None:
            return w
        n, r, k = w.shape
        return (w.view(n, r // 128, 128, k // 128, 128) * scales[experts][:, :, None, :, None]).view(n, r, k)

    up = s["x"].float()[None] @ wide(s["w13"], s["s13"]).transpose(1, 2)  # [active, T, 2 I]
    inter = up.size(2) // 2
    gate = up[..., :inter]
    hidden = gate / (1.0 + torch.exp(-gate)) * up[..., inter:] * share.sum(-1)[..., None]
    return (hidden @ wide(s["w2"], s["s2"]).transpose(1, 2)).sum(0).to(torch.bfloat16)


def _plain_norm(s):
    """total = x + residual; y = total * weight / sqrt(mean(total^2) + eps); q, scales: e4m3 with one scale per 128 channels of the normed row."""
    total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(torch.bfloat16)
    t, w = total.float(), s["weight"].float()
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    y = t * r * w
    if not s["train"]:
        blocks = y.view(y.size(0), -1, 128)
        amax = blocks.abs().amax(-1, keepdim=True).clamp(min=1e-4)
        q = (blocks * (448.0 / amax)).view(y.shape).to(torch.float8_e4m3fn)
        return dict(q=q, scales=(amax / 448.0).squeeze(-1), y=y.to(torch.bfloat16), total=None if s["residual"] is None else total)
    dy = s["dy"].float()
    wdy = w * dy
    gx = r * (wdy - t * r * r * (wdy * t).mean(-1, keepdim=True))
    gw = (dy * t * r).sum(0).to(s["weight"].dtype)
    if s["residual"] is None:
        return dict(y=y.to(torch.bfloat16), total=None, gx=gx.to(torch.bfloat16), gr=None, gw=gw)
    gx = (gx + s["ds"].float()).to(torch.bfloat16)
    return dict(y=y.to(torch.bfloat16), total=total, gx=gx, gr=gx, gw=gw)


def _plain_route(s):
    """The k largest logits, the lowest index first among equals; weights: softmax over them, or over all experts. An expert with -inf is none (-1, weight 0)."""
    logits = s["logits"].float()
    values, idx = torch.sort(logits, dim=-1, descending=True, stable=True)
    values, idx = values[:, : s["topk"]], idx[:, : s["topk"]]
    taken = values != -math.inf
    idx = torch.where(taken, idx, torch.full_like(idx, -1))
    top = torch.where(taken[:, :1], values[:, :1], torch.zeros_like(values[:, :1]))
    e = torch.exp((values if s["renormalize"] else logits) - top)
    total = e.sum(-1, keepdim=True).clamp(min=1e-38)
    weights = torch.exp(values - top) / total
    if s["dw"] is None:
        return dict(idx=idx, weights=weights, dlogits=None)
    inner = (s["dw"] * weights).sum(-1, keepdim=True)
    base = torch.zeros_like(logits) if s["renormalize"] else -inner * e / total
    own_part = weights * (s["dw"] - inner) if s["renormalize"] else weights * s["dw"]
    dlogits = base.scatter_add(1, idx.clamp(min=0), torch.where(taken, own_part, torch.zeros_like(own_part)))
    return dict(idx=idx, weights=weights, dlogits=dlogits.to(s["logits"].dtype))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------
def work(case):
    c, T = case, case["tokens"]
    if c["kind"] == "experts":
        H, inter, each = c["hidden"], c["inter"], 1 if c["fp8"] else 2
        k = c["topk"] * (1.0 - c["dropped"])
        active = c["local"] * (1.0 - (1.0 - k / c["experts"]) ** T)  # experts that some token chose, on average
        pairs = T * k * c["local"] / c["experts"]
        scales = 4 * 3 * H * inter // 128 // 128 if c["fp8"] else 0
        return dict(bytes=active * (3 * H * inter * each + scales) + 4 * T * H + 12 * T * c["topk"], flops=6.0 * H * inter * pairs)
    if c["kind"] == "norm":
        H, rows = c["hidden"], T * c["hidden"]
        r = 1 if c["residual"] else 0
        weight = H * (4 if c["wide"] else 2)
        if not c["train"]:
            return dict(bytes=rows * (2 + 2 * r + 2 * r + 2 + 1) + rows // 128 * 4 + weight, flops=6.0 * rows)
        return dict(bytes=rows * ((2 + 2 * r + 2 * r + 2) + (2 + 2 * r + 2)) + 2 * weight, flops=16.0 * rows)
    E, each = c["experts"], 2 if c["bf16"] else 4
    n = T * E
    if not c["train"]:
        return dict(bytes=n * each + T * c["topk"] * 12, flops=2.0 * n)
    return dict(bytes=2 * n * each + T * c["topk"] * 16, flops=6.0 * n)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "experts":
        x, out = s["x"].double(), torch.zeros(s["x"].shape, dtype=torch.float64, device=DEVICE)
        ids, share = s["idx"].tolist(), s["weights"].double()
        inter = s["w2"].size(2)

        def wide(w, scales, e):
            w = w[e].double()
            return w if scales is None else w * scales[e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)

        for e in range(s["w13"].size(0)):
            at = [(t, k) for t, row in enumerate(ids) for k, i in enumerate(row) if i == e + s["first"]]
            if not at:
                continue
            t, k = (torch.tensor(v, device=DEVICE) for v in zip(*at))
            both = x[t] @ wide(s["w13"], s["s13"], e).T
            a, b = both[:, :inter], both[:, inter:]
            out.index_add_(0, t, ((a * torch.sigmoid(a) * b) @ wide(s["w2"], s["s2"], e).T) * share[t, k][:, None])
        return out
    if s["kind"] == "norm":
        # the sum is rounded to the stream's type by definition; the quotients of q are given before their rounding
        total = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        t = (s["x"] if s["residual"] is None else total.float().to(torch.bfloat16)).double().requires_grad_(True)
        w = s["weight"].double().requires_grad_(True)
        y = t * w / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS)
        kept = None if s["residual"] is None else total
        if not s["train"]:
            v = y.detach().unflatten(-1, (-1, 128))
            scale = v.abs().amax(-1).clamp(min=1e-4) / 448.0
            return dict(q=(v / scale[..., None]).flatten(1), scales=scale, y=y.detach(), total=kept)
        gt, gw = torch.autograd.grad((y * s["dy"].double()).sum() + (0.0 if s["ds"] is None else (t * s["ds"].double()).sum()), (t, w))
        return dict(y=y.detach(), total=kept, gx=gt, gr=None if s["residual"] is None else gt, gw=gw)
    logits = s["logits"].double().requires_grad_(True)
    order = torch.argsort(logits.detach(), dim=-1, descending=True, stable=True)[:, : s["topk"]]
    values = logits.gather(1, order)
    gone = values.detach() == -math.inf
    norm = torch.logsumexp(values if s["renormalize"] else logits, -1, keepdim=True)
    weights = torch.where(gone, torch.zeros_like(values), torch.exp(values - norm))
    idx = order.masked_fill(gone, -1)
    if s["dw"] is None:
        return dict(idx=idx, weights=weights.detach(), dlogits=None)
    (dl,) = torch.autograd.grad((weights * s["dw"].double()).sum(), logits)
    return dict(idx=idx, weights=weights.detach(), dlogits=torch.nan_to_num(dl))
