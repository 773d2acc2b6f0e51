"""Norm, choice of the experts and experts for a few tokens on the GPU, against 64 bits (tolerances: block_refs.py), and the block that runs them."""
import pytest
import torch

import block_refs as refs

pytestmark = pytest.mark.gpu


def _ops():
    from deepep_efa_b200.ops import few_tokens, norm, router
    return norm.rms_norm, norm.rms_norm_fp8, router.select_experts, few_tokens.few_token_experts


def _rows(n, h, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, h, generator=g, device="cuda") * std).to(torch.bfloat16)


def _weight(h, wide, seed=9):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (1 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(torch.float32 if wide else torch.bfloat16)


# ---- norm -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,h", [(1, 8), (1, 7168), (2, 32768), (3, 72), (149, 264), (700, 1032), (333, 2056), (301, 4096), (160, 6152), (155, 7168), (150, 9000), (149, 18776)])
@pytest.mark.parametrize("wide,residual", [(False, True), (True, False), (True, True)])
def test_norm_and_its_gradients(n, h, wide, residual):
    rms_norm = _ops()[0]
    x, r, dy, dt, w = _rows(n, h, 1).requires_grad_(), _rows(n, h, 2, 3.0).requires_grad_(), _rows(n, h, 3), _rows(n, h, 4), _weight(h, wide).requires_grad_()
    if residual:
        y, total = rms_norm(x, w, r)
        assert torch.equal(total.detach(), (x + r).detach())
        grads = torch.autograd.grad((y, total), (x, r, w), (dy, dt))
        assert torch.equal(grads[0], grads[1])
    else:
        y, total, dt = rms_norm(x, w), x, None
        grads = torch.autograd.grad(y, (x, w), dy)
    exact, _ = refs.norm(total.detach(), w.detach(), 1e-6)
    assert ((y.double() - exact).abs() <= (refs.BF16 + refs.NORM) * exact.abs()).all()
    dx, x_bound, dw, w_bound = refs.norm_gradients(total.detach(), w.detach(), dy, dt, 1e-6)
    assert grads[-1].dtype == w.dtype
    assert ((grads[0].double() - dx).abs() <= x_bound).all() and ((grads[-1].double() - dw).abs() <= w_bound).all()


@pytest.mark.parametrize("n,h", [(1, 128), (1, 7168), (5, 384), (400, 4096), (200, 7168), (150, 16384)])
@pytest.mark.parametrize("round_scale", [False, True])
def test_norm_with_fp8_rows(n, h, round_scale):
    rms_norm, rms_norm_fp8 = _ops()[:2]
    x, r, w = _rows(n, h, 5), _rows(n, h, 6), _weight(h, True)
    x[0, :128] = 0
    r[0, :128] = 0
    (q, s), y, total = rms_norm_fp8(x, w, r, round_scale=round_scale)
    y2, total2 = rms_norm(x, w, r)
    assert torch.equal(y, y2) and torch.equal(total, total2)
    exact, _ = refs.norm(total, w, 1e-6)
    scale = s.double().repeat_interleave(128, 1)
    assert ((q.double() * scale - exact).abs() <= (refs.E4M3 + refs.NORM) * exact.abs() + 2.0 ** -10 * scale).all()
    amax = exact.abs().view(n, -1, 128).amax(-1).clamp(min=1e-4) / 448
    if round_scale:
        assert torch.equal(s, torch.exp2(torch.round(torch.log2(s))))
        assert (s.double() >= amax * (1 - 2 * refs.NORM)).all() and (s.double() < 2 * amax * (1 + 2 * refs.NORM)).all()
    else:
        assert torch.allclose(s.double(), amax, rtol=2 * refs.NORM, atol=0)
    (q3, s3), y3, none = rms_norm_fp8(total, w, round_scale=round_scale, keep_rows=False)
    assert y3 is None and none is None and torch.equal(q3.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s3, s)


def test_norm_of_other_layouts():
    """Rows of a wider matrix, of one that has to be copied, three dimensions, no rows, the gradient of a sum (one number for all), only one of two outputs used."""
    rms_norm = _ops()[0]
    w = _weight(256, False).requires_grad_()
    wide = _rows(50, 1024, 7)
    for x in (wide[:, 256:512], wide[:, 3:259], wide.t()[:256, :].t()[:, :256], wide[::2, :256], wide[:1, :256].expand(9, 256)):
        y, total = rms_norm(x, w, x)
        y2, total2 = rms_norm(x.contiguous(), w, x.contiguous())
        assert torch.equal(y, y2) and torch.equal(total, total2)
    three = wide[:, :768].reshape(50, 3, 256)
    y, total = rms_norm(three, w, three)
    assert y.shape == three.shape and torch.equal(y.view(-1, 256), rms_norm(three.reshape(-1, 256), w, three.reshape(-1, 256))[0])
    x = wide[:, :256].clone().requires_grad_()
    y, total = rms_norm(x, w, x)
    (alone,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    (same,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    assert torch.equal(alone, same)
    past = torch.autograd.grad(total, (x, w), torch.full_like(total, 2.0), allow_unused=True)
    assert (past[0] == 4).all() and past[1] is None
    empty = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y, total = rms_norm(empty, w, empty)
    gx, gw = torch.autograd.grad((y, total), (empty, w), (y, total))
    assert gx.shape == (0, 256) and (gw == 0).all()


def test_norm_of_rows_out_of_the_ordinary():
    """Zeros, numbers whose squares are no floats, infinities and NaN: each stays in its row."""
    rms_norm, rms_norm_fp8 = _ops()[:2]
    x = _rows(200, 512, 8)
    x[3] = 0
    x[5, 7] = float("inf")
    x[6, 9] = float("nan")
    w = _weight(512, True)
    y = rms_norm(x, w)
    (q, s), y8, _ = rms_norm_fp8(x, w)
    fine = [i for i in range(200) if i not in (5, 6)]
    exact, _ = refs.norm(x[fine], w, 1e-6)
    assert ((y[fine].double() - exact).abs() <= (refs.BF16 + refs.NORM) * exact.abs()).all() and (y[3] == 0).all() and (q[3].float() == 0).all()
    assert torch.isnan(y[5, 7]) and torch.isnan(y[6]).all() and torch.isnan(q[6].float()).all()
    assert torch.equal(y8[fine], y[fine])


def test_norm_gradients_repeat_and_are_captured():
    """Bit for bit from run to run; forward and backward captured into a graph and replayed on other inputs, on a stream of its own."""
    rms_norm = _ops()[0]
    x, r, dy, dt, w = _rows(900, 4096, 1), _rows(900, 4096, 2), _rows(900, 4096, 3), _rows(900, 4096, 4), _weight(4096, True)

    def step():
        a, b, c = x.detach().requires_grad_(), r.detach().requires_grad_(), w.detach().requires_grad_()
        y, total = rms_norm(a, c, b)
        return (y.detach(), total.detach(), *torch.autograd.grad((y, total), (a, b, c), (dy, dt)))
    first = step()
    assert all(torch.equal(p, q) for p, q in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (11, 12):
        x.copy_(_rows(900, 4096, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_norm_refusals():
    rms_norm, rms_norm_fp8 = _ops()[:2]
    x, w = _rows(4, 256, 1), _weight(256, True)
    for bad in (lambda: rms_norm(x.float(), w), lambda: rms_norm(x[:, :252], w[:252]), lambda: rms_norm(x, w[:128]), lambda: rms_norm(x, w.double()), lambda: rms_norm(x, w.cpu()),
                lambda: rms_norm(x, w, x[:2]), lambda: rms_norm(x, w, x.float()), lambda: rms_norm(x, w, x.cpu()), lambda: rms_norm_fp8(x[:, :136], w[:136]),
                lambda: rms_norm(torch.zeros(1, 32776, dtype=torch.bfloat16, device="cuda"), torch.ones(32776, device="cuda")),
                lambda: rms_norm_fp8(x.clone().requires_grad_(), w)):
        with pytest.raises(ValueError):
            bad()


# ---- choice of the experts ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,n,k", [(1, 1, 1), (3, 8, 8), (257, 60, 4), (1000, 64, 6), (513, 160, 6), (700, 256, 8), (65, 1000, 32), (5, 1024, 7)])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_choice_and_its_gradient(tokens, n, k, renormalize, dtype):
    select_experts = _ops()[2]
    g = torch.Generator(device="cuda").manual_seed(n + k)
    logits = (2 * torch.randn(tokens, n, generator=g, device="cuda")).to(dtype)
    logits[torch.rand(tokens, n, generator=g, device="cuda") < 0.1] = -torch.inf
    logits[:1] = -torch.inf
    if tokens > 2:
        logits[1] = 0.25
        logits[2, ::2] = 0.0
        logits[2, 1::2] = -0.0
    logits = logits.requires_grad_()
    idx, weights = select_experts(logits, k, renormalize=renormalize)
    want, exact = refs.select(logits.detach(), k, renormalize)
    assert torch.equal(idx, want) and (weights[idx < 0] == 0).all() and idx.dtype == torch.int64 and weights.dtype == torch.float32
    # exp of a difference that is rounded once, two units of expf, under 48 additions, a division
    values = logits.detach().double().gather(1, want.clamp(min=0))
    top = values[:, :1].clamp(min=-1e30)
    rel = (56 + (values - top).abs().clamp(max=1e3)) * 2.0 ** -24
    ok = want >= 0
    assert ((weights.double() - exact).abs() <= rel * exact)[ok].all()
    dw = torch.randn(tokens, k, generator=g, device="cuda")
    (dl,) = torch.autograd.grad(weights, logits, dw)
    l64 = logits.detach().double().requires_grad_()
    some = ok.any(-1)
    v64 = l64.gather(1, want.clamp(min=0)).masked_fill(~ok, -torch.inf)
    w64 = torch.exp(v64 - torch.logsumexp(v64 if renormalize else l64, -1, keepdim=True))
    d64 = torch.zeros_like(l64)
    if some.any():
        (d64,) = torch.autograd.grad((w64[some] * dw.double()[some]).sum(), l64)
    d64 = d64.nan_to_num()  # (a row without experts has no gradient)
    # weights as above; the sum over k products and the differences: k + 4 roundings of terms of at most |g| and sum |w g|
    most = dw.double().abs().amax(-1, keepdim=True)
    p = torch.softmax(l64.detach(), -1).nan_to_num()
    p = torch.maximum(p, torch.zeros_like(p).scatter_reduce_(1, want.clamp(min=0), exact.masked_fill(~ok, 0.0), "amax"))
    bound = 2 * (80 + k + 40) * 2.0 ** -24 * most * p + (refs.BF16 * d64.abs() if dtype == torch.bfloat16 else 0)
    assert dl.dtype == dtype and ((dl.double() - d64).abs() <= bound + 1e-30).all()
    assert (dl[~some] == 0).all()


def test_choice_gradient_is_its_differences():
    """Central differences of the kernel's own weights: h^2 / 6 times the third derivative (at most 1/4 per weight), and the weights' 2^-18 over h."""
    select_experts = _ops()[2]
    g = torch.Generator(device="cuda").manual_seed(3)
    logits, dw, h = torch.randn(4, 10, generator=g, device="cuda"), torch.randn(4, 3, generator=g, device="cuda"), 2.0 ** -6
    for renormalize in (False, True):
        leaf = logits.clone().requires_grad_()
        idx, weights = select_experts(leaf, 3, renormalize=renormalize)
        (dl,) = torch.autograd.grad(weights, leaf, dw)
        for e in range(10):
            plus, minus = logits.clone(), logits.clone()
            plus[:, e] += h
            minus[:, e] -= h
            (ip, wp), (im, wm) = select_experts(plus, 3, renormalize=renormalize), select_experts(minus, 3, renormalize=renormalize)
            same = ((ip == idx) & (im == idx)).all(-1)
            diff = ((wp - wm).double() * dw.double()).sum(-1) / (2 * h)
            tol = dw.double().abs().sum(-1) * (h * h / 6 / 4 + 2.0 ** -18 / h)
            assert ((diff - dl[:, e].double()).abs() <= tol)[same].all()


def test_choice_of_logits_out_of_the_ordinary():
    select_experts = _ops()[2]
    logits = torch.zeros(4, 40, device="cuda")
    logits[0, 7] = float("nan")
    logits[1, 9] = float("inf")
    logits[2, 33] = -float("nan")
    idx, weights = select_experts(logits, 3)
    assert idx[0].tolist() == [7, 0, 1] and idx[1].tolist() == [9, 0, 1] and idx[2].tolist() == [33, 0, 1] and idx[3].tolist() == [0, 1, 2]
    assert torch.isnan(weights[0]).all() and torch.isnan(weights[2]).all() and (weights[3] - 1 / 3).abs().max() < 2.0 ** -22
    wide = torch.randn(100, 96, device="cuda")
    for part in (wide[:, 10:74], wide[::3, :64], wide.t()[:64].t(), wide[:1, :64].expand(50, 64)):
        assert all(torch.equal(p, q) for p, q in zip(select_experts(part, 4), select_experts(part.contiguous(), 4)))
    none = select_experts(torch.empty(0, 8, device="cuda"), 2)
    assert none[0].shape == (0, 2) and none[1].shape == (0, 2)


def test_choice_refusals():
    select_experts = _ops()[2]
    x = torch.zeros(3, 16, device="cuda")
    for bad in (lambda: select_experts(x, 0), lambda: select_experts(x, 17), lambda: select_experts(x.half(), 2), lambda: select_experts(x[0], 2),
                lambda: select_experts(torch.zeros(3, 64, device="cuda"), 33), lambda: select_experts(torch.zeros(3, 1025, device="cuda"), 2),
                lambda: select_experts(torch.zeros(3, 0, device="cuda"), 1)):
        with pytest.raises(ValueError):
            bad()


# ---- experts for a few tokens -----------------------------------------------------------------------------------------------------------
def _check(v, y, first=0):
    out, bound = refs.experts(*v, first=first)
    assert y.dtype == torch.bfloat16 and ((y.double() - out).abs() <= bound).all(), ((y.double() - out).abs() / bound).max().item()
    return out


@pytest.mark.parametrize("tokens,hidden,inter,local,topk,total,dropped", [
    (1, 256, 128, 4, 2, None, 0.0), (1, 2048, 1408, 8, 6, None, 0.0), (2, 1024, 256, 8, 1, None, 0.5), (3, 1152, 640, 16, 4, 24, 0.2), (8, 512, 384, 12, 8, None, 0.0),
    (9, 512, 128, 3, 2, None, 0.0), (16, 640, 256, 5, 5, None, 0.0), (17, 384, 256, 40, 8, 80, 0.1), (32, 256, 128, 2, 2, None, 0.0), (32, 512, 256, 64, 8, 128, 0.0)])
@pytest.mark.parametrize("fp8", [False, True])
def test_experts(tokens, hidden, inter, local, topk, total, dropped, fp8):
    few = _ops()[3]
    v = refs.layer_inputs(tokens, hidden, inter, local, topk, fp8, "cuda", seed=tokens + hidden, experts_total=total, dropped=dropped)
    first = (total or local) - local
    y = few(*v[:5], w13_scales=v[5], w2_scales=v[6], first_expert=first)
    _check(v, y, first)
    assert torch.equal(y, few(*v[:5], w13_scales=v[5], w2_scales=v[6], first_expert=first))


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 8, 8), (5, 72, 24), (3, 1032, 648), (7, 1000, 40), (32, 136, 1416)])
def test_experts_of_ragged_widths(tokens, hidden, inter):
    few = _ops()[3]
    v = refs.layer_inputs(tokens, hidden, inter, 6, 3, False, "cuda", seed=inter)
    _check(v, few(*v[:5]))


@pytest.mark.parametrize("fp8", [False, True])
def test_experts_of_selections_out_of_the_ordinary(fp8):
    """Nobody's expert here, the same expert several times for a token, all tokens on one expert, one expert that many ids name (more than one group), top-32."""
    few = _ops()[3]
    x, idx, weights, w13, w2, s13, s2 = refs.layer_inputs(32, 256, 128, 8, 4, fp8, "cuda", seed=1)
    run = lambda i, w, n=32, **k: few(x[:n], i[:n], w[:n], w13, w2, w13_scales=s13, w2_scales=s2, **k)  # noqa: E731
    assert (run(torch.full_like(idx, -1), weights) == 0).all() and (run(idx, weights, first_expert=100) == 0).all() and (run(idx, weights, first_expert=-100) == 0).all()
    assert run(idx, weights, n=0).shape == (0, 256)
    for n in (1, 2, 9, 32):
        for i in (torch.full_like(idx, 5), idx % 2, torch.stack([idx[:, 0], idx[:, 1], idx[:, 0], idx[:, 0]], 1)):
            y = run(i, weights, n)
            _check((x[:n], i[:n], weights[:n], w13, w2, s13, s2), y)
    many = torch.arange(32, device="cuda").repeat(32, 1) % 10 - 1
    share = torch.rand(32, 32, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    y = few(x, many, share, w13, w2, w13_scales=s13, w2_scales=s2)
    _check((x, many, share, w13, w2, s13, s2), y)
    big = torch.full_like(idx, 2 ** 40)
    big[0, 0] = 3
    _check((x, big, weights, w13, w2, s13, s2), run(big, weights))


@pytest.mark.parametrize("fp8", [False, True])
def test_experts_of_numbers_out_of_the_ordinary(fp8):
    """Tokens of very different size side by side, zeros, an outlier within a token, NaN and infinities in one token, weights of zero and below."""
    few = _ops()[3]
    v = refs.layer_inputs(6, 512, 256, 4, 2, fp8, "cuda", seed=3)
    x, weights = v[0], v[2]
    x[0] *= 1e-6
    x[1] *= 1e3
    x[2] = 0
    x[3, 100] = 300
    weights[4, 0] = 0
    weights[5, 1] = -2.5
    run = lambda: few(*v[:5], w13_scales=v[5], w2_scales=v[6])  # noqa: E731
    y = run()
    _check(v, y)
    assert (y[2] == 0).all()
    for bad in (float("nan"), float("inf")):
        x[3, 7] = bad
        z = run()
        keep = [0, 1, 2, 4, 5]
        assert torch.equal(z[keep], y[keep]) and not torch.isfinite(z[3].float()).all()
    if fp8:  # a weight that is no number reaches the results of its expert's tokens and no others
        x[3] = 1
        w13 = v[3].view(torch.uint8)
        w13[2, 5, 9] = 0x7F
        z = run()
        hit = (v[1] == 2).any(-1)
        assert torch.isnan(z[hit].float()).all() and torch.isfinite(z[~hit].float()).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_experts_among_many(fp8):
    """The most experts there may be; the last one's weights end the tensor."""
    few = _ops()[3]
    v = refs.layer_inputs(32, 128, 128, 1024, 32, fp8, "cuda", seed=4)
    v[1][0, 0], v[1][1, 1] = 1023, 0
    _check(v, few(*v[:5], w13_scales=v[5], w2_scales=v[6]))


def test_experts_of_other_layouts_and_streams():
    """Rows of a wider matrix, transposed ids, weights that only a stream's earlier work writes, several streams at once, a captured step replayed on other inputs and
    routing, and rows behind the result's left as they were."""
    few = _ops()[3]
    v = refs.layer_inputs(5, 512, 256, 8, 2, False, "cuda", seed=5)
    x, idx, weights, w13, w2 = v[:5]
    y = few(x, idx, weights, w13, w2)
    wide = torch.zeros(5, 2048, dtype=torch.bfloat16, device="cuda")
    wide[:, 512:1024] = x
    assert torch.equal(few(wide[:, 512:1024], idx.t().contiguous().t(), weights.t().contiguous().t(), w13, w2), y)
    odd = torch.zeros(5, 515, dtype=torch.bfloat16, device="cuda")
    odd[:, 3:] = x
    assert torch.equal(few(odd[:, 3:], idx, weights, w13, w2), y)
    room = torch.full((8, 512), 3.0, dtype=torch.bfloat16, device="cuda")
    few(x, idx, weights, w13, w2, out=room[:5])
    assert torch.equal(room[:5], y) and (room[5:] == 3).all()
    other = refs.layer_inputs(32, 512, 256, 8, 8, False, "cuda", seed=6)
    want = few(*other[:3], w13, w2)
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append((few(x, idx, weights, w13, w2), y) if i else (few(*other[:3], w13, w2), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
    graphs = []
    for n in (5, 3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = few(x[:n], idx[:n], weights[:n], w13, w2)
        graphs.append((graph, out, n))
    for seed in (7, 8):
        for a, b in zip((x, idx, weights), refs.layer_inputs(5, 512, 256, 8, 2, False, "cuda", seed=seed, dropped=0.3)):
            a.copy_(b)
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        # (a token's sums are taken in an order that goes by all experts of the batch: the same batch, the same bits)
        assert all(torch.equal(out, few(x[:n], idx[:n], weights[:n], w13, w2)) for _, out, n in graphs)


def test_experts_refusals():
    few = _ops()[3]
    x, idx, weights, w13, w2, s13, s2 = refs.layer_inputs(4, 256, 128, 4, 2, True, "cuda")
    b13, b2 = w13.to(torch.bfloat16), w2.to(torch.bfloat16)
    ok = dict(w13_scales=s13, w2_scales=s2)
    for bad in (lambda: few(x.float(), idx, weights, w13, w2, **ok), lambda: few(x, idx.int(), weights, w13, w2, **ok), lambda: few(x, idx, weights.double(), w13, w2, **ok),
                lambda: few(x, idx, weights[:3], w13, w2, **ok), lambda: few(x, idx[:3], weights[:3], w13, w2, **ok), lambda: few(x, idx, weights, w13, w2),
                lambda: few(x, idx, weights, b13, b2, **ok), lambda: few(x, idx, weights, w13, b2, **ok), lambda: few(x, idx, weights, w13, w2, w13_scales=s13, w2_scales=s2[:, :1]),
                lambda: few(x, idx, weights, w13[:, :, :128], w2, **ok), lambda: few(x, idx, weights, b13[:, 1:], b2), lambda: few(x, idx, weights, b13, b2[:3]),
                lambda: few(x, idx, weights, b13.transpose(1, 2), b2.transpose(1, 2)), lambda: few(x, idx, weights, b13.cpu(), b2), lambda: few(x, idx.cpu(), weights, b13, b2),
                lambda: few(x, idx, weights, b13, b2, out=torch.empty(4, 256, device="cuda")), lambda: few(x, idx, weights, b13, b2, out=torch.empty(3, 256, device="cuda", dtype=torch.bfloat16)),
                lambda: few(x[:, :132], idx, weights, b13[:, :, :132].contiguous(), b2[:, :132].contiguous()), lambda: few(x.repeat(9, 1), idx.repeat(9, 1), weights.repeat(9, 1), b13, b2),
                lambda: few(x, torch.zeros(4, 33, dtype=torch.int64, device="cuda"), torch.zeros(4, 33, device="cuda"), b13, b2),
                lambda: few(x.clone().requires_grad_(), idx, weights, b13, b2)):
        with pytest.raises(ValueError):
            bad()


# ---- together ---------------------------------------------------------------------------------------------------------------------------
def test_block():
    """The three as a block of one rank: training with gradients, FP8 prefill whose dispatch takes the norm's rows, decode of a few tokens eagerly and from a graph, two
    blocks one after the other."""
    from deepep_efa_b200 import _ext
    from deepep_efa_b200.models.moe import MoEBlock, MoEConfig, dense_reference
    from deepep_efa_b200.parallel.virtual import VirtualCluster
    rms_norm, rms_norm_fp8, select_experts, _ = _ops()
    H, inter, E, K = 512, 256, 16, 4
    vc = VirtualCluster(1, num_nvl_bytes=64 << 20, num_rdma_bytes=0)
    rel = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()  # noqa: E731
    try:
        buf = vc.buffers[0]
        blocks = [MoEBlock(MoEConfig(hidden=H, intermediate=inter, num_experts=E, num_topk=K, init_std=0.05), buf, seed=s) for s in (1, 2)]
        x, r = _rows(20, H, 1).requires_grad_(), _rows(20, H, 2).requires_grad_()
        y, total = blocks[0](x, r)
        (y.float().square().mean() + total.float().mean()).backward()
        torch.cuda.synchronize()
        buf.check_status()
        b = blocks[0]
        assert all(p.grad is not None and torch.isfinite(p.grad.float()).all() and (p.grad != 0).any() for p in (x, r, b.norm, b.moe.gate, b.moe.w13, b.moe.w2))
        normed, kept = rms_norm(x.detach(), b.norm.detach(), r.detach())
        idx, weights = b.moe.choose(normed)
        i2, w2 = b.moe.route(normed)
        assert torch.equal(idx, i2) and (weights - w2).abs().max() < 2.0 ** -18
        ref = dense_reference(normed, idx, weights, b.moe.w13.detach().float(), b.moe.w2.detach().float())
        assert torch.equal(total, kept) and rel(y, ref) < 3e-2
        few, few_total = b.forward_few_tokens(x.detach(), r.detach(), fp8=False)
        assert torch.equal(few_total, kept) and rel(few, ref) < 1e-2
        for native in (True, False):
            b.moe.prepare_fp8(native_block_scaling=native)
            rows, normed2, _ = rms_norm_fp8(x.detach(), b.norm.detach(), r.detach(), round_scale=native)
            y8, total8 = b.forward_fp8(x.detach(), r.detach())
            assert torch.equal(normed2, normed) and torch.equal(total8, kept) and rel(y8, ref) < 8e-2
            assert torch.equal(y8, b.moe.forward_fp8(rows, idx, weights))
            # rows that the caller cast are those that the dispatch casts
            cast = _ext.load().per_token_cast_to_fp8(normed, native, False)
            assert torch.equal(b.moe.forward_fp8(cast, idx, weights), b.moe.forward_fp8(normed, idx, weights))
            buf.check_status()
            f8, _ = b.forward_few_tokens(x.detach(), r.detach())
            assert rel(f8, ref) < 5e-2
            # next to the quantised weights themselves the form for a few tokens keeps its own accuracy
            (q13, s13), (q2, s2) = b.moe._fp8
            out, bound = refs.experts(normed, idx, weights, q13, q2, s13, s2)
            assert ((f8.double() - out).abs() <= bound).all()
        with pytest.raises(ValueError):
            b.moe.forward_fp8(rows)
        # a decode step through both blocks, captured
        def step(x, r):
            for block in blocks:
                x, r = block.forward_few_tokens(x, r)
            return x, r
        xs, rs = x.detach().clone()[:3], r.detach().clone()[:3]
        step(xs, rs)
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            out = step(xs, rs)
        for seed in (5, 6):
            xs.copy_(_rows(3, H, seed))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, step(xs, rs)))
        assert _ext.load().gemm_error(0) == 0
    finally:
        vc.destroy()


def test_few_tokens_need_every_expert():
    """A rank that holds a part of the experts is told to use the exchange."""
    from deepep_efa_b200.models.moe import MoEConfig, MoELayer
    from deepep_efa_b200.parallel.virtual import VirtualCluster
    vc = VirtualCluster(2, num_nvl_bytes=8 << 20, num_rdma_bytes=0)
    try:
        layer = MoELayer(MoEConfig(hidden=128, intermediate=128, num_experts=4, num_topk=2), vc.buffers[0])
        with pytest.raises(ValueError, match="forward_low_latency"):
            layer.forward_few_tokens(_rows(2, 128, 1))
    finally:
        vc.destroy()


def test_rows_far_apart():
    """Rows whose last one begins past 2^31 elements: the norm and its gradients, the choice, the experts' tokens."""
    rms_norm, _, select_experts, few = _ops()
    room = torch.empty(300, 2 ** 23, dtype=torch.bfloat16, device="cuda")
    parts = [room[:, at:at + 256] for at in (8, 512, 1024, 2048)]
    for i, part in enumerate(parts):
        part.copy_(_rows(300, 256, 20 + i))
    w = _weight(256, True)
    near = [p.contiguous() for p in parts]

    def step(x, r, dy, dt):
        x, r, c = x.detach().requires_grad_(), r.detach().requires_grad_(), w.detach().requires_grad_()
        y, total = rms_norm(x, c, r)
        return (y.detach(), total.detach(), *torch.autograd.grad((y, total), (x, r, c), (dy, dt)))
    assert all(torch.equal(p, q) for p, q in zip(step(*parts), step(*near)))
    assert all(torch.equal(p, q) for p, q in zip(select_experts(parts[0], 8), select_experts(near[0], 8)))
    _, idx, weights, w13, w2, _, _ = refs.layer_inputs(32, 256, 64, 4, 2, False, "cuda")
    assert torch.equal(few(parts[0][268:], idx, weights, w13, w2), few(near[0][268:], idx, weights, w13, w2))


def test_experts_captured_first():
    """A capture before anything else of the library ran on the device: its error word is not the graph's."""
    import os
    import subprocess
    import sys
    code = ("import torch, block_refs as refs; from deepep_efa_b200 import _ext; from deepep_efa_b200.ops.few_tokens import few_token_experts as few\n"
            "v = refs.layer_inputs(3, 128, 128, 4, 2, True, 'cuda'); _ext.load(); torch.cuda.synchronize(); g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n    y = few(*v[:5], w13_scales=v[5], w2_scales=v[6])\n"
            "g.replay(); torch.cuda.synchronize(); out, bound = refs.experts(*v)\n"
            "assert ((y.double() - out).abs() <= bound).all() and _ext.load().gemm_error(0) == 0; print('fine')")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join((root, os.path.join(root, "tests"))))
    done = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]
