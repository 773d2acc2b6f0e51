"""What stands around the experts of a block where numbers or calls are out of the ordinary, without a GPU."""
import types

import pytest
import torch

import block_refs as refs
from deepep_efa_b200 import _ext
from deepep_efa_b200.models.moe import MoEConfig, MoELayer
from deepep_efa_b200.ops.norm import rms_norm, rms_norm_fp8


class Reached(Exception):
    pass


def lone_layer():
    """A layer of a lone rank whose buffer says that it was reached."""
    def layout(*_):
        raise Reached
    buffer = types.SimpleNamespace(group_size=1, rank=0, get_dispatch_layout=layout)
    return MoELayer(MoEConfig(hidden=256, intermediate=128, num_experts=4, num_topk=2), buffer, device=torch.device("cpu"))


# ---- a copy that does not come --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("stages", [2, 3])
@pytest.mark.parametrize("boxes", [0, 1, 2, 3, 4, 7, 12])
def test_ring_of_a_warp_whose_wait_runs_out(stages, boxes):
    """The kernels' loop over a warp's boxes with the wait for each of them, or for none, running out: the copies that are still on their way are waited for, each in its
    slot with the parity of its use, once; nothing is started after that."""
    for fails_at in range(boxes + 1):
        ring, todo, flying, uses = _ext.load().FewTokensRing(stages), list(range(boxes)), [], [0] * stages

        def start():
            if todo:
                assert all(slot != ring.fill for slot, _ in flying)  # (a slot is filled when its box has been read)
                flying.append((ring.fill, uses[ring.fill] & 1))
                uses[ring.fill] += 1
                todo.pop(0)
                ring.started()
        for _ in range(stages):
            start()
        waits = []
        for box in range(boxes):
            if box >= fails_at:  # (the CTA's flag ends every wait from then on)
                ring.give_up(lambda slot, parity: waits.append((slot, parity)))
                assert not ring.alive and waits == flying and len(waits) == min(stages, boxes - fails_at)
            else:
                assert (ring.slot, ring.parity) == flying.pop(0)
            assert 0 <= ring.slot < stages
            ring.taken()
            if ring.alive:
                start()
                assert ring.flying == len(flying)
        assert ring.alive == (fails_at == boxes) and (not ring.alive or not flying) and ring.flying <= 0


# ---- quantised rows and native block scaling ----------------------------------------------------------------------------------------------
def test_quantised_rows_need_the_layers_scales():
    """Native block scaling reads a scale's exponent alone: rows whose scales are no powers of two, or are not said to be, do not get as far as the dispatch."""
    layer, w = lone_layer(), torch.ones(256)
    layer.prepare_fp8(native_block_scaling=False)
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    idx, weights = torch.zeros(5, 2, dtype=torch.int64), torch.ones(5, 2)
    plain, powers = rms_norm_fp8(x, w)[0], rms_norm_fp8(x, w, round_scale=True)[0]
    for rows in (plain, powers, (plain[0], plain[1].t().contiguous().t())):
        for said in (None, False, True):  # fp32 scales of any kind
            with pytest.raises(Reached):
                layer.forward_fp8(rows, idx, weights, round_scale=said)
    layer._mx = ()
    for rows, said in ((powers, None), (powers, True), ((powers[0], powers[1].t().contiguous().t()), None), ((powers[0][:0], powers[1][:0]), None), (x, None)):
        with pytest.raises(Reached):
            layer.forward_fp8(rows, idx, weights, round_scale=said)
    one = powers[1].clone()
    one[3, 1] *= 1 + 2.0 ** -23
    for rows, said in ((plain, None), (powers, False), ((powers[0], one), None)):
        with pytest.raises(ValueError, match="powers of two"):
            layer.forward_fp8(rows, idx, weights, round_scale=said)
    with pytest.raises(ValueError, match="expert ids"):
        layer.forward_fp8(powers)


# ---- rows whose squares are no floats ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("wide", [False, True])
def test_norm_of_large_rows(wide):
    """Rows from 2^10 to the largest bf16 beside ordinary ones: the norm does not depend on a row's size, and neither do the bounds."""
    g = torch.Generator().manual_seed(7)
    x, dy, dt = (torch.randn(40, 256, generator=g).to(torch.bfloat16) for _ in range(3))
    for i, power in enumerate((10, 30, 39, 40, 41, 42, 58, 59, 60, 61, 63, 64, 80, 120, 124)):
        x[2 * i] *= 2.0 ** power
    x[39, 1:], x[39, 0] = 0, 3e38
    dt[::4] = 0
    x.requires_grad_()
    w = (1 + 0.2 * torch.randn(256, generator=g)).to(torch.float32 if wide else torch.bfloat16).requires_grad_()
    y, total = rms_norm(x, w, torch.zeros_like(x))
    exact, _ = refs.norm(x.detach(), w.detach(), 1e-6)
    assert torch.equal(total, x) and ((y.double() - exact).abs() <= (refs.BF16 + refs.NORM) * exact.abs()).all()
    gx, gw = torch.autograd.grad((y, total), (x, w), (dy, dt))
    dx, x_bound, dw, w_bound = refs.norm_gradients(x.detach(), w.detach(), dy, dt, 1e-6)
    # (a gradient below bf16's normal numbers is off by half of its smallest step)
    assert ((gx.double() - dx).abs() <= x_bound + 2.0 ** -134).all() and ((gw.double() - dw).abs() <= w_bound).all()
    (q, s), y8, _ = rms_norm_fp8(x.detach(), w.detach())
    scale = s.double().repeat_interleave(128, 1)
    assert torch.equal(y8, y) and ((q.double() * scale - exact).abs() <= (refs.E4M3 + refs.NORM) * exact.abs() + 2.0 ** -10 * scale).all()
