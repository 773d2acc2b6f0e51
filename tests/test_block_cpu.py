"""Norm, choice of the experts and experts for a few tokens on CPU tensors, against 64 bits; what they refuse; a block of all three over gloo."""
import os
import socket

import pytest
import torch

import block_refs as refs
from deepep_efa_b200.ops.few_tokens import few_token_experts
from deepep_efa_b200.ops.norm import rms_norm, rms_norm_fp8
from deepep_efa_b200.ops.router import select_experts


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_norm_and_its_gradients(residual, wide):
    g = torch.Generator().manual_seed(1)
    x, r, dy, dt = (torch.randn(5, 136, generator=g).to(torch.bfloat16) for _ in range(4))
    w = (1 + 0.2 * torch.randn(136, generator=g)).to(torch.float32 if wide else torch.bfloat16)
    x, r, w = x.requires_grad_(), r.requires_grad_(), w.requires_grad_()
    if residual:
        y, total = rms_norm(x, w, r)
        assert torch.equal(total, (x + r))
        grads = torch.autograd.grad((y, total), (x, r, w), (dy, dt))
        assert torch.equal(grads[0], grads[1])
    else:
        total, dt = x, None
        y = rms_norm(x, w)
        grads = torch.autograd.grad(y, (x, w), dy)
    exact, _ = refs.norm(total.detach(), w.detach(), 1e-6)
    assert ((y.double() - exact).abs() <= (refs.BF16 + refs.NORM) * exact.abs()).all()
    dx, x_bound, dw, w_bound = refs.norm_gradients(total.detach(), w.detach(), dy, dt, 1e-6)
    assert ((grads[0].double() - dx).abs() <= x_bound).all() and ((grads[-1].double() - dw).abs() <= w_bound).all()


def test_gradients_of_the_norm_are_its_differences():
    """The formulas that the kernels are held to, against central differences of the forward formula, both in 64 bits: the error of a difference over 2 h is
    h^2 / 6 times the third derivative, here below 100, and 2^-53 of the sum over h."""
    g = torch.Generator().manual_seed(2)
    t, w, dy = (torch.randn(3, 24, generator=g, dtype=torch.float64) for _ in range(3))
    w = w[0]
    dx, _, dw, _ = refs.norm_gradients(t, w, dy, None, 1e-6)
    h = 1e-4
    loss = lambda t, w: (refs.norm(t, w, 1e-6)[0] * dy).sum()  # noqa: E731
    for i in range(24):
        e = torch.zeros(24, dtype=torch.float64)
        e[i] = h
        at = torch.zeros_like(t)
        at[1, i] = h
        assert abs((loss(t + at, w) - loss(t - at, w)) / (2 * h) - dx[1, i]) < 1e-6
        assert abs((loss(t, w + e) - loss(t, w - e)) / (2 * h) - dw[i]) < 1e-6


@pytest.mark.parametrize("round_scale", [False, True])
def test_norm_with_fp8_rows(round_scale):
    g = torch.Generator().manual_seed(3)
    x, r = (torch.randn(4, 256, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(256)
    (q, s), y, total = rms_norm_fp8(x, w, r, round_scale=round_scale)
    exact, _ = refs.norm(total, w, 1e-6)
    scale = s.double().repeat_interleave(128, 1)
    assert ((q.double() * scale - exact).abs() <= (refs.E4M3 + refs.NORM) * exact.abs() + 2.0 ** -10 * scale).all()
    if round_scale:
        assert torch.equal(s, torch.exp2(torch.round(torch.log2(s))))
    assert rms_norm_fp8(x, w, keep_rows=False)[1:] == (None, None)


@pytest.mark.parametrize("renormalize", [False, True])
def test_choice_and_its_gradient(renormalize):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(9, 12, generator=g).to(torch.bfloat16).float()
    logits[0] = 1.0
    logits[1] = -torch.inf
    logits[2, :10] = -torch.inf
    logits = logits.requires_grad_()
    idx, weights = select_experts(logits, 4, renormalize=renormalize)
    want, exact = refs.select(logits.detach(), 4, renormalize)
    assert torch.equal(idx, want) and idx[0].tolist() == [0, 1, 2, 3] and idx[1].tolist() == [-1] * 4 and (weights[1] == 0).all()
    assert torch.allclose(weights.double()[2:], exact[2:], rtol=2.0 ** -18, atol=0)
    dw = torch.randn(9, 4, generator=g)
    (dl,) = torch.autograd.grad(weights, logits, dw)
    l64 = logits.detach().double().requires_grad_()
    rows = [r for r in range(9) if r != 1]
    values = l64.gather(1, want.clamp(min=0)).masked_fill(want < 0, -torch.inf)
    w64 = torch.exp(values - torch.logsumexp(values if renormalize else l64, -1, keepdim=True))
    (d64,) = torch.autograd.grad((w64[rows] * dw.double()[rows]).sum(), l64)
    assert torch.allclose(dl.double()[rows], d64[rows], rtol=0, atol=2.0 ** -18 * float(dw.abs().max()) * 4)
    assert (dl[1] == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_experts(fp8):
    x, idx, weights, w13, w2, s13, s2 = refs.layer_inputs(7, 256, 128, 6, 3, fp8, "cpu", experts_total=9, dropped=0.2)
    y = few_token_experts(x, idx, weights, w13, w2, w13_scales=s13, w2_scales=s2, first_expert=2)
    out, bound = refs.experts(x, idx, weights, w13, w2, s13, s2, first=2)
    assert ((y.double() - out).abs() <= bound).all()
    into = torch.full_like(x, 7.0)
    assert few_token_experts(x, idx, weights, w13, w2, w13_scales=s13, w2_scales=s2, first_expert=2, out=into) is into and torch.equal(into, y)


def test_refusals():
    x, idx, weights, w13, w2, _, _ = refs.layer_inputs(33, 64, 32, 4, 2, False, "cpu")
    with pytest.raises(ValueError, match="32 tokens"):
        few_token_experts(x, idx, weights, w13, w2)
    with pytest.raises(ValueError, match="forward only"):
        few_token_experts(x[:2], idx[:2], weights[:2], w13.requires_grad_(), w2)
    with torch.no_grad():
        few_token_experts(x[:2], idx[:2], weights[:2], w13, w2)
    with pytest.raises(ValueError, match="weight must be"):
        rms_norm(x, torch.ones(63))
    with pytest.raises(ValueError, match="residual must be"):
        rms_norm(x, torch.ones(64), x[:3])
    with pytest.raises(ValueError, match="multiple of 128"):
        rms_norm_fp8(x, torch.ones(64))
    with pytest.raises(ValueError, match="forward only"):
        rms_norm_fp8(x.clone().requires_grad_(), torch.ones(64))
    for k in (0, 5, 33):
        with pytest.raises(ValueError, match="num_topk"):
            select_experts(torch.zeros(2, 4), k)


def test_block_over_gloo():
    """Norm, choice and layer as a block: forward, gradients, and the form for a few tokens with the same weights."""
    import torch.distributed as dist

    import deepep_efa_b200 as ep
    from deepep_efa_b200.models.moe import MoEBlock, MoEConfig, dense_reference
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        buf = ep.Buffer(dist.group.WORLD, num_nvl_bytes=1 << 20)
        block = MoEBlock(MoEConfig(hidden=64, intermediate=128, num_experts=8, num_topk=2, init_std=0.1), buf, device=torch.device("cpu"))
        g = torch.Generator().manual_seed(5)
        x, r = (torch.randn(6, 64, generator=g).to(torch.bfloat16).requires_grad_() for _ in range(2))
        y, total = block(x, r)
        (y.float().square().mean() + total.float().mean()).backward()
        assert all(p.grad is not None and torch.isfinite(p.grad.float()).all() for p in (x, r, block.norm, block.moe.gate, block.moe.w13, block.moe.w2))
        normed, kept = rms_norm(x.detach(), block.norm.detach(), r.detach())
        idx, weights = block.moe.route(normed)
        ref = dense_reference(normed, idx, weights, block.moe.w13.detach().float(), block.moe.w2.detach().float())
        few, few_total = block.forward_few_tokens(x.detach(), r.detach(), fp8=False)
        assert torch.equal(few_total, total) and torch.equal(few_total, kept)
        rel = lambda a, b: ((a.float() - b.float()).norm() / b.float().norm()).item()  # noqa: E731
        assert rel(y, ref) < 3e-2 and rel(few, ref) < 1e-2
    finally:
        dist.destroy_process_group()
