"""Norm, choice of the experts and experts for a few tokens on the GPU where numbers, gradients or calls are out of the ordinary (tolerances: block_refs.py)."""
import types

import pytest
import torch

import block_refs as refs
from deepep_efa_b200.ops.few_tokens import few_token_experts
from deepep_efa_b200.ops.norm import rms_norm, rms_norm_fp8
from deepep_efa_b200.ops.router import select_experts

pytestmark = pytest.mark.gpu


# ---- weights that are no numbers ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [2, 6, 32])
@pytest.mark.parametrize("fp8", [False, True])
def test_experts_keep_a_bad_w2_to_its_tokens(tokens, fp8):
    """NaN and infinity in one expert's W2 (or its scales) reach the results of this expert's tokens, in the rows that hold them, and nothing else: every other number
    is that of finite weights, bit for bit. Experts have groups of different size, one after the other in a warp's run of boxes."""
    x, idx, weights, w13, w2, s13, s2 = refs.layer_inputs(tokens, 512, 384, 7, 3, fp8, "cuda", seed=tokens)
    idx[0] = torch.tensor([2, 3, 5], device="cuda")
    idx[1:] = torch.where(idx[1:] == 2, torch.full_like(idx[1:], -1), idx[1:])  # expert 2 has one token, the next ones have more
    run = lambda w2, s2: few_token_experts(x, idx, weights, w13, w2, w13_scales=s13, w2_scales=s2)  # noqa: E731
    good = run(w2, s2)
    cases = []
    for e in range(7):
        if fp8:
            bad = w2.clone()
            bad.view(torch.uint8)[e, 9, ::64] = 0x7F
            cases.append((e, bad, s2, slice(9, 10)))
            for v in (float("nan"), float("inf")):
                scales = s2.clone()
                scales[e, 1] = v
                cases.append((e, w2, scales, slice(128, 256)))
        else:
            for v in (float("nan"), float("inf")):
                bad = w2.clone()
                bad[e, 9, ::64] = v
                cases.append((e, bad, s2, slice(9, 10)))
    for e, w, s, rows in cases:
        y, hit = run(w, s), (idx == e).any(-1)
        assert not torch.isfinite(y[hit][:, rows].float()).any()
        keep = torch.ones(512, dtype=torch.bool, device="cuda")
        keep[rows] = False
        assert torch.equal(y[~hit], good[~hit]) and torch.equal(y[:, keep], good[:, keep]), (e, int((y[~hit] != good[~hit]).sum()))


# ---- small values beside zeros ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 6])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, 1e-8])
def test_experts_with_rows_of_zeros(tokens, size):
    """Sixteen gate rows, sixteen up rows, or all but sixteen, that are zero (pruned, or padded to the multiple of 128) cost the others of their box nothing."""
    for zero in (slice(0, 16), slice(112, 128), slice(384 + 32, 384 + 48), slice(16, 384)):
        v = refs.layer_inputs(tokens, 256, 384, 4, 2, True, "cuda", seed=11)
        v[0] *= size
        v[3].view(torch.uint8)[:, zero] = 0
        y = few_token_experts(*v[:5], w13_scales=v[5], w2_scales=v[6])
        out, bound = refs.experts(*v)
        assert ((y.double() - out).abs() <= bound).all(), ((y.double() - out).abs() / bound).max().item()


# ---- infinite hidden values ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
def test_experts_with_an_infinite_hidden_value(fp8):
    """gate * up past the largest float is an infinity, which the result has with the sign of its weight, whatever finite values of any size stand beside it; and
    values between the largest bf16 and the largest float stay finite."""
    H, inter = 128, 256
    x = torch.zeros(2, H, dtype=torch.bfloat16, device="cuda")
    x[0, 0] = x[1, 0] = 1e19
    w13, w2 = torch.zeros(1, 2 * inter, H, device="cuda"), torch.zeros(1, H, inter, device="cuda")
    w13[0, :, 0] = 2.0 ** -4         # (6e17)^2
    w13[0, [40, inter + 40], 0] = 2  # (2e19)^2: infinite
    w2[0] = -1
    w2[0, :, 40] = 1
    w2[0, ::2] *= -1
    one = torch.ones(2, 1, device="cuda")
    idx = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    if fp8:
        scales = dict(w13_scales=torch.ones(1, 2 * inter // 128, H // 128, device="cuda"), w2_scales=torch.ones(1, H // 128, inter // 128, device="cuda"))
        a, b = w13.to(torch.float8_e4m3fn), w2.to(torch.float8_e4m3fn)
    else:
        scales, a, b = {}, w13.to(torch.bfloat16), w2.to(torch.bfloat16)
    y = few_token_experts(x, idx, one, a, b, **scales).float()
    assert (y[:, 0::2] == -torch.inf).all() and (y[:, 1::2] == torch.inf).all()
    # one value alone, 2^128 (1 - 2^-10): a bf16 rounding of it would be infinite
    w13.zero_()
    w2.zero_()
    w13[0, [3, inter + 3], 0] = 1
    w2[0, :, 3] = 2.0 ** -6
    x[:, 0] = 2.0 ** 63
    a, b = w13.to(a.dtype), w2.to(b.dtype)
    y = few_token_experts(x, idx, one * (4 * (1 - 2.0 ** -10)), a, b, **scales).double()
    exact = 2.0 ** 122 * (1 - 2.0 ** -10)
    assert ((y - exact).abs() <= (refs.BF16 + 2.0 ** -10) * exact).all()


# ---- gradient of a choice that has a NaN --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_choice_gradient_with_nan(dtype):
    """Probabilities among all experts are NaN in a row with a NaN, and so is every entry of its gradient; among the chosen ones, theirs. As on the CPU."""
    logits = torch.randn(6, 40, generator=torch.Generator().manual_seed(1)).to(dtype)
    logits[1, 7] = float("nan")
    logits[2, 9] = float("inf")
    logits[3, 5] = -float("inf")
    logits[4, 5], logits[4, 30] = -float("inf"), float("nan")
    dw = torch.randn(6, 3, generator=torch.Generator().manual_seed(2))
    for renormalize in (False, True):
        def gradient(device):
            leaf = logits.to(device).requires_grad_()
            _, weights = select_experts(leaf, 3, renormalize=renormalize)
            return torch.autograd.grad(weights, leaf, dw.to(device))[0].cpu()
        here, there = gradient("cuda"), gradient("cpu")
        assert torch.equal(torch.isnan(here), torch.isnan(there))
        if not renormalize:
            assert torch.isnan(here[[1, 2, 4]]).all()
        assert torch.isfinite(here[[0, 3, 5]].float()).all()


# ---- quantised rows and native block scaling ----------------------------------------------------------------------------------------------
def test_quantised_rows_need_the_layers_scales():
    """Native block scaling reads a scale's exponent alone. Rows whose scales are no powers of two are refused, found by looking or by what the caller says of them."""
    from deepep_efa_b200.models.moe import MoEBlock, MoEConfig
    from deepep_efa_b200.parallel.virtual import VirtualCluster
    vc = VirtualCluster(1, num_nvl_bytes=64 << 20, num_rdma_bytes=0)
    try:
        block = MoEBlock(MoEConfig(hidden=256, intermediate=256, num_experts=8, num_topk=2, init_std=0.05), vc.buffers[0])
        layer, w = block.moe, block.norm.detach()
        x = torch.randn(40, 256, device="cuda").to(torch.bfloat16)
        for native in (True, False):
            layer.prepare_fp8(native_block_scaling=native)
            (plain, y, _), (powers, _, _) = rms_norm_fp8(x, w), rms_norm_fp8(x, w, round_scale=True)
            with torch.no_grad():
                idx, weights = layer.choose(y)
            want = layer.forward_fp8(y, idx, weights)
            assert torch.equal(layer.forward_fp8(powers, idx, weights), layer.forward_fp8(powers, idx, weights, round_scale=True))
            if native:
                assert torch.equal(layer.forward_fp8(powers, idx, weights), block.forward_fp8(x)[0])
                with pytest.raises(ValueError, match="powers of two"):
                    layer.forward_fp8(plain, idx, weights)
                with pytest.raises(ValueError, match="powers of two"):
                    layer.forward_fp8(powers, idx, weights, round_scale=False)
            else:
                assert torch.equal(layer.forward_fp8(plain, idx, weights), block.forward_fp8(x)[0])
            assert torch.isfinite(want.float()).all()
        vc.buffers[0].check_status(sync=True)
    finally:
        vc.destroy()


# ---- tangents -----------------------------------------------------------------------------------------------------------------------------
def test_forward_mode_is_refused():
    """A tangent is not dropped without a word."""
    import torch.autograd.forward_ad as fwd
    x, w = torch.randn(4, 128, device="cuda").to(torch.bfloat16), torch.ones(128, device="cuda")
    logits = torch.randn(4, 8, device="cuda")
    v = refs.layer_inputs(3, 128, 128, 4, 2, False, "cuda")
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for bad in (lambda: rms_norm(dual(x), w), lambda: rms_norm(x, dual(w)), lambda: rms_norm(x, w, dual(x)), lambda: rms_norm_fp8(dual(x), w), lambda: rms_norm_fp8(x, w, dual(x)),
                    lambda: select_experts(dual(logits), 2), lambda: few_token_experts(dual(v[0]), *v[1:5]), lambda: few_token_experts(*v[:2], dual(v[2]), *v[3:5]),
                    lambda: few_token_experts(*v[:4], dual(v[4]))):
            with pytest.raises(NotImplementedError):
                bad()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                bad()
        rms_norm(x, w), select_experts(logits, 2), few_token_experts(*v[:5])


# ---- second derivatives -------------------------------------------------------------------------------------------------------------------
def test_second_derivatives_are_refused():
    """Gradients that were asked for with a graph have one that says so; those that need none are as ever."""
    x, w = torch.randn(4, 128, device="cuda").to(torch.bfloat16).requires_grad_(), torch.ones(128, device="cuda", requires_grad=True)
    dy = torch.randn(4, 128, device="cuda").to(torch.bfloat16)
    for residual in (None, x):
        out = rms_norm(x, w, residual)
        y = out if residual is None else out[0]
        plain = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        kept = torch.autograd.grad(y, (x, w), dy, create_graph=True)
        assert all(torch.equal(a, b.detach()) and not a.requires_grad and b.requires_grad for a, b in zip(plain, kept))
        for g, leaf in ((kept[0], x), (kept[0], w), (kept[1], x)):
            with pytest.raises(RuntimeError, match="differentiable"):
                torch.autograd.grad(g.float().square().sum(), leaf, retain_graph=True)
        # beside a term that is twice differentiable it would be lost in silence
        with pytest.raises(RuntimeError, match="differentiable"):
            ((kept[0].float() + x.float().square()).sum()).backward(inputs=[x])
        with pytest.raises(RuntimeError, match="differentiable"):
            torch.autograd.grad((kept[1].float() + w.square()).sum(), w, retain_graph=True)
    _, total = rms_norm(x, w, x)
    (past,) = torch.autograd.grad(total, x, dy, create_graph=True)  # (a sum alone is linear)
    assert torch.equal(past.detach(), dy + dy)
    logits = torch.randn(5, 8, device="cuda", requires_grad=True)
    for renormalize in (False, True):
        _, weights = select_experts(logits, 2, renormalize=renormalize)
        dw = torch.randn(5, 2, device="cuda")
        plain, kept = (torch.autograd.grad(weights, logits, dw, retain_graph=True, create_graph=c)[0] for c in (False, True))
        assert torch.equal(plain, kept.detach())
        with pytest.raises(RuntimeError, match="differentiable"):
            torch.autograd.grad(kept.square().sum(), logits)


# ---- a result in a tensor that a graph has kept ----------------------------------------------------------------------------------------------
def test_experts_into_a_tensor_that_was_kept_for_a_gradient():
    v = refs.layer_inputs(3, 128, 128, 4, 2, False, "cuda")
    out, leaf = torch.ones(3, 128, dtype=torch.bfloat16, device="cuda"), torch.ones(3, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    kept = (out * leaf).sum()
    few_token_experts(*v[:5], out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    with pytest.raises(ValueError, match="forward only"):
        few_token_experts(*v[:5], out=leaf)
    with torch.inference_mode():
        few_token_experts(*v[:5], out=torch.empty(3, 128, dtype=torch.bfloat16, device="cuda"))


# ---- weights that are quantised on the way -------------------------------------------------------------------------------------------------
def test_few_tokens_are_not_captured_before_the_weights_are_quantised():
    """Weights quantised inside a capture would hold nothing until its first replay, and be quantised again by each."""
    from deepep_efa_b200.models.moe import MoEBlock, MoEConfig
    buffer = types.SimpleNamespace(group_size=1, rank=0)
    block = MoEBlock(MoEConfig(hidden=128, intermediate=128, num_experts=4, num_topk=2), buffer, device=torch.device("cuda"))
    x = torch.randn(3, 128, device="cuda").to(torch.bfloat16)
    block.forward_few_tokens(x, fp8=False)  # (what libraries make on their first call)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="prepare_fp8"):
        with torch.cuda.graph(graph):
            block.forward_few_tokens(x)
    assert block.moe._fp8 is None
    want = block.forward_few_tokens(x)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block.forward_few_tokens(x)[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ---- rows whose squares are no floats ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("h", [128, 1032, 7168, 12000, 20000])
@pytest.mark.parametrize("wide", [False, True])
def test_norm_of_large_rows(h, wide):
    """Rows from 2^10 to the largest bf16 beside ordinary ones: the norm does not depend on a row's size, and neither do the bounds."""
    g = torch.Generator(device="cuda").manual_seed(h)
    x, dy, dt = ((torch.randn(170, h, generator=g, device="cuda")).to(torch.bfloat16) for _ in range(3))
    for i, power in enumerate((10, 20, 30, 38, 39, 40, 41, 42, 50, 57, 58, 59, 60, 61, 62, 63, 64, 65, 80, 100, 120, 124)):
        x[5 * i] *= 2.0 ** power
    x[169, 1:], x[169, 0] = 0, 3e38
    dt[::2] = 0
    x.requires_grad_()
    w = (1 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(torch.float32 if wide else torch.bfloat16).requires_grad_()
    y, total = rms_norm(x, w, torch.zeros_like(x))
    exact, _ = refs.norm(x.detach(), w.detach(), 1e-6)
    assert torch.equal(total, x) and ((y.double() - exact).abs() <= (refs.BF16 + refs.NORM) * exact.abs()).all()
    alone = rms_norm(x, w)
    assert torch.equal(alone, y)
    gx, gw = torch.autograd.grad((y, total), (x, w), (dy, dt), retain_graph=True)
    dx, x_bound, dw, w_bound = refs.norm_gradients(x.detach(), w.detach(), dy, dt, 1e-6)
    # (a gradient below bf16's normal numbers is off by half of its smallest step)
    assert ((gx.double() - dx).abs() <= x_bound + 2.0 ** -134).all(), ((gx.double() - dx).abs() / (x_bound + 2.0 ** -134)).max().item()
    assert ((gw.double() - dw).abs() <= w_bound).all()
    (gx,) = torch.autograd.grad(alone, x, dy)
    dx, x_bound, _, _ = refs.norm_gradients(x.detach(), w.detach(), dy, None, 1e-6)
    assert ((gx.double() - dx).abs() <= x_bound + 2.0 ** -134).all()
    if h % 128 == 0:
        (q, s), y8, _ = rms_norm_fp8(x.detach(), w.detach())
        scale = s.double().repeat_interleave(128, 1)
        assert torch.equal(y8, y) and ((q.double() * scale - exact).abs() <= (refs.E4M3 + refs.NORM) * exact.abs() + 2.0 ** -10 * scale).all()


@pytest.mark.parametrize("rows,h", [(100, 2048), (100, 7168), (600, 264), (600, 2048), (600, 4096)])
def test_norm_of_rows_that_are_large_in_parts(rows, h):
    """Rows whose warps lie on both sides of where squares are summed in another scale: all of them count."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(rows, h, generator=g, device="cuda")
    x *= 2.0 ** torch.linspace(45, 51, rows, device="cuda")[:, None]
    half = (torch.arange(h, device="cuda") // 256) % 2 == 0  # (a warp's channels, where a thread has eight)
    x[::2, half] *= 0.5
    x, w = x.to(torch.bfloat16), torch.ones(h, device="cuda")
    y = rms_norm(x, w)
    exact, _ = refs.norm(x, w, 1e-6)
    assert ((y.double() - exact).abs() <= (refs.BF16 + refs.NORM) * exact.abs()).all()
