"""The choice of a token's experts from its gate logits (kernels in csrc/kernels/router.cu).

The reference leaves routing to its users; the ids and weights made here are what ``Buffer.dispatch`` and ``MoELayer`` take.
"""
from __future__ import annotations

from typing import Tuple

import torch

from .. import _ext


class _SelectExperts(torch.autograd.Function):
    """The CPU form."""

    @staticmethod
    def forward(ctx, logits, num_topk, renormalize):
        ctx.renormalize = renormalize
        ctx.set_materialize_grads(False)
        if logits.dim() != 2 or not 1 <= num_topk <= min(32, logits.size(1)) or logits.size(1) > 1024:
            raise ValueError("deepep_efa_b200.select_experts: logits must be [T, E], num_topk 1 to 32 and at most E, E at most 1024")
        values, order = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
        values, order = values[:, :num_topk], order[:, :num_topk]
        gone = values == -torch.inf
        idx = order.masked_fill(gone, -1)
        top = values[:, :1].masked_fill(gone[:, :1], 0.0)
        total = torch.exp((values if renormalize else logits.float()) - top).sum(-1, keepdim=True)
        weights = torch.where(gone, torch.zeros_like(values), torch.exp(values - top) / total)
        ctx.mark_non_differentiable(idx)
        ctx.save_for_backward(logits, idx, weights)
        return idx, weights

    @staticmethod
    def backward(ctx, _, dweights):
        if dweights is None:
            return None, None, None
        logits, idx, weights = ctx.saved_tensors
        chosen = idx >= 0
        inner = torch.where(chosen, weights * dweights, torch.zeros_like(weights)).sum(-1, keepdim=True)
        dlogits = torch.zeros(logits.shape, dtype=torch.float32) if ctx.renormalize else -inner * torch.softmax(logits.float(), -1).nan_to_num()
        at = torch.where(chosen, weights * dweights - (weights * inner if ctx.renormalize else 0.0), torch.zeros_like(weights))
        return dlogits.scatter_add_(1, idx.clamp(min=0), at).to(logits.dtype), None, None


def select_experts(logits: torch.Tensor, num_topk: int, *, renormalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(topk_idx int64, topk_weights fp32)``, both ``[T, num_topk]``, for gate logits ``[T, E]`` in fp32 or bf16 (``E`` up to 1024, ``num_topk`` up to 32).

    A token gets its ``num_topk`` largest logits in falling order, of equal ones the lowest index first, NaN before all others. Weights are the softmax over the
    chosen logits, or with ``renormalize=False`` their probabilities among all experts. An expert whose logit is ``-inf`` is not chosen: what then is left over of
    a row is ``-1`` with weight 0 (dispatch skips it). Differentiable in ``logits``."""
    if not logits.is_cuda:
        return _SelectExperts.apply(logits, num_topk, renormalize)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _ext.load().select_experts_grad(logits, num_topk, renormalize)
    return _ext.load().select_experts(logits, num_topk, renormalize)
