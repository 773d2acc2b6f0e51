"""A layer of routed SwiGLU experts for a few tokens, without dispatch and combine (kernels in csrc/kernels/few_tokens.cu).

A decode step of up to 32 tokens whose experts are on this GPU is bound by reading the chosen experts' weights; this form does little else. The reference
is a communication library and has no counterpart; users of its low-latency pair run the experts between dispatch and combine.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _ext

MAX_TOKENS = 32


def few_token_experts(x: torch.Tensor, topk_idx: torch.Tensor, topk_weights: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, *,
                      w13_scales: Optional[torch.Tensor] = None, w2_scales: Optional[torch.Tensor] = None, first_expert: int = 0,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_k topk_weights[t, k] * w2[e] @ (silu(gate[e] @ x[t]) * (up[e] @ x[t]))`` with ``e = topk_idx[t, k] - first_expert``; bf16 ``[T, H]``.

    ``x`` bf16 ``[T, H]``, ``T`` up to 32; ``topk_idx`` int64 and ``topk_weights`` fp32 ``[T, K]``. ``w13`` ``[L, 2 I, H]`` holds gate above up, ``w2`` is ``[L, H, I]``: bf16
    (``H``, ``I`` multiples of 8), or e4m3 with fp32 scales per block of 128 x 128 (``MoELayer.prepare_fp8``; multiples of 128). Sums are in fp32. Hidden values, their
    weights included, are kept as two bf16 numbers (16 bits) next to bf16 weights, as fp16 with a power of two per 16 values (11 bits; 2^-24 of the largest of 128) next
    to e4m3 ones, where ``x`` too is fp16 over a power of two per token (exact to 2^-17 of a token's largest magnitude, off by at most 2^-25 of it below). Ids without
    an expert in ``[first_expert, first_expert + L)`` are skipped, so ranks that share the experts each compute their part of the sum. Forward only; no host
    synchronisation, so a step can be captured into a graph. A copy that does not come within two seconds ends the call with a wrong result and sets the
    device's error word, which ``Buffer.check_status(sync=True)`` reads (a capture before any other call of the library on that device has none)."""
    if x.is_cuda:
        return _ext.load().few_tokens(x, topk_idx, topk_weights, w13, w2, w13_scales, w2_scales, first_expert, out)
    if torch.is_grad_enabled() and (x.requires_grad or topk_weights.requires_grad or w13.requires_grad or w2.requires_grad):
        raise ValueError("deepep_efa_b200.few_token_experts: forward only; call it under torch.no_grad()")
    if x.size(0) > MAX_TOKENS:
        raise ValueError("deepep_efa_b200.few_token_experts: at most 32 tokens")
    y = reference_few_token_experts(x, topk_idx, topk_weights, w13, w2, w13_scales, w2_scales, first_expert).to(x.dtype)
    return y if out is None else out.copy_(y)


def reference_few_token_experts(x, topk_idx, topk_weights, w13, w2, w13_scales=None, w2_scales=None, first_expert=0, dtype=torch.float32) -> torch.Tensor:
    """Plain PyTorch form of :func:`few_token_experts` in ``dtype``, one expert after the other (CPU tensors, tests)."""
    def wide(w, scales, e):
        return w[e].to(dtype) if scales is None else w[e].to(dtype) * scales[e].to(dtype).repeat_interleave(128, 0).repeat_interleave(128, 1)

    out = torch.zeros(x.shape, dtype=dtype, device=x.device)
    inter = w2.size(2)
    for e in range(w13.size(0)):
        t, k = (topk_idx == e + first_expert).nonzero(as_tuple=True)
        if t.numel() == 0 or e + first_expert < 0:
            continue
        both = x[t].to(dtype) @ wide(w13, w13_scales, e).t()
        h = torch.nn.functional.silu(both[:, :inter]) * both[:, inter:]
        out.index_add_(0, t, (h @ wide(w2, w2_scales, e).t()) * topk_weights[t, k].to(dtype).unsqueeze(1))
    return out
