"""Root-mean-square norm of the residual stream in front of a block of experts (kernels in csrc/kernels/norm.cu).

    total = x + residual                        rounded to the stream's bf16
    y     = total * weight / sqrt(mean(total ** 2) + eps)

``rms_norm`` has gradients; ``rms_norm_fp8`` is for serving and also gives the normed rows as ``(e4m3, fp32 scales per 128 channels)``, the form that
``Buffer.dispatch`` and ``MoELayer.forward_fp8`` take. CPU tensors are computed by PyTorch operations, so that a layer runs under gloo.

The reference library has no model code and so no counterpart.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _ext


def _total(x: torch.Tensor, residual: Optional[torch.Tensor]) -> torch.Tensor:
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def _check_cpu(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor]) -> None:
    if weight.dim() != 1 or weight.size(0) != x.size(-1):
        raise ValueError("deepep_efa_b200.rms_norm: weight must be [H]")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("deepep_efa_b200.rms_norm: residual must be of x's shape and type")


def _sized(t: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(rows, 1 / sqrt(mean square + eps) of them, the power of two that they were multiplied with)``: large rows, whose squares are no floats, are made small first."""
    down = torch.where(t.abs().amax(-1, keepdim=True) > 2.0 ** 40, 2.0 ** -80, 1.0)
    t = t * down
    return t, torch.rsqrt(t.square().mean(-1, keepdim=True) + eps * down * down), down


class _RMSNorm(torch.autograd.Function):
    """The CPU form."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.eps, ctx.has_residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        _check_cpu(x, weight, residual)
        total = None if residual is None else _total(x, residual)
        t, r, _ = _sized((x if residual is None else total).float(), eps)
        y = (t * r * weight.float()).to(x.dtype)
        ctx.save_for_backward(x if residual is None else total, weight)
        return y if residual is None else (y, total)

    @staticmethod
    def backward(ctx, dy, dtotal=None):
        total, weight = ctx.saved_tensors
        if dy is None:
            dx, dw = dtotal, None
        else:
            (t, r, down), g = _sized(total.float(), ctx.eps), dy.float()
            wg = g * weight.float()
            dx = down * (r * (wg - t * r * r * (wg * t).mean(-1, keepdim=True)))
            dx = (dx if dtotal is None else dx + dtotal.float()).to(total.dtype)
            dw = (g * t * r).sum(0).to(weight.dtype)
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """The norm of the rows of ``x`` (bf16 ``[..., H]``, ``H`` a multiple of 8 up to 32768; ``weight`` bf16 or fp32 ``[H]``). Returns ``y``, or with a ``residual``
    of ``x``'s shape ``(y, x + residual)``. A row's size does not matter, up to the largest bf16. Differentiable in all three, once; ``weight``'s gradient is summed in fp32 in a fixed order and has its type."""
    shape = x.shape
    if x.dim() != 2:
        if residual is not None and residual.shape != shape:
            raise ValueError("deepep_efa_b200.rms_norm: residual must be of x's shape")
        x, residual = x.reshape(-1, shape[-1]), None if residual is None else residual.reshape(-1, shape[-1])
    if x.is_cuda:
        out = _ext.load().rms_norm_grad(x, weight, residual, eps)
    else:
        out = _RMSNorm.apply(x, weight, residual, eps)
        out = (out,) if residual is None else out
    if len(shape) != 2:
        out = [o.view(shape) for o in out]
    return out[0] if residual is None else (out[0], out[1])


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6, round_scale: bool = False,
                 keep_rows: bool = True) -> Tuple[Tuple[torch.Tensor, torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The norm for serving (no gradients): ``((q, scales), y, total)`` for bf16 ``x`` ``[N, H]``, ``H`` a multiple of 128.

    ``q`` e4m3 ``[N, H]`` and ``scales`` fp32 ``[N, H / 128]`` are made from the normed values in fp32 as the dispatch casts its rows (largest magnitude of 128
    channels, at least 1e-4, over 448; with ``round_scale`` rounded up to a power of two). ``y`` is bf16, None without ``keep_rows``; ``total`` is None without ``residual``."""
    if x.is_cuda:
        return _ext.load().rms_norm_fp8(x, weight, residual, eps, round_scale, keep_rows)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        raise ValueError("deepep_efa_b200.rms_norm_fp8: forward only; call it under torch.no_grad()")
    _check_cpu(x, weight, residual)
    if x.dim() != 2 or x.size(1) % 128 != 0:
        raise ValueError("deepep_efa_b200.rms_norm_fp8: x must be [N, H] with H a multiple of 128")
    total = _total(x, residual)
    t, r, _ = _sized(total.float(), eps)
    v = t * r * weight.float()
    amax = v.view(v.size(0), -1, 128).abs().amax(-1).clamp(min=1e-4)
    scales, inv = amax / 448.0, 448.0 / amax
    if round_scale:
        scales = torch.exp2(torch.ceil(torch.log2(scales)))
        inv = 1.0 / scales
    q = (v.view(v.size(0), -1, 128) * inv.unsqueeze(-1)).view(v.shape).to(torch.float8_e4m3fn)
    return (q, scales), v.to(x.dtype) if keep_rows else None, None if residual is None else total
