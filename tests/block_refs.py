"""What the norm, the choice of experts and the experts for a few tokens compute, in 64 bits, with how far the kernels may be off.

Rounding to a type is off by half a step: bf16 2^-8, fp16 2^-11, e4m3 2^-4 of the value (2^-10 of its scale below e4m3's normal numbers)."""
import torch

BF16, FP16, E4M3 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -4
# Sums of a norm: a thread adds at most 32 numbers, then a tree over a warp and at most 32 warps: under 80 additions deep, of which half the relative error reaches the root.
NORM = 80 * 2.0 ** -24


def norm(total, weight, eps):
    """y and 1 / sqrt(mean square + eps) of rows in 64 bits."""
    t = total.double()
    r = 1.0 / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
    return t * r * weight.double(), r


def norm_gradients(total, weight, dy, dtotal, eps):
    """(dx, its bound, dweight, its bound) by the formulas."""
    t, w, g = total.double(), weight.double(), dy.double()
    _, r = norm(total, weight, eps)
    inner = (w * g * t).mean(-1, keepdim=True)
    direct, back, past = r * w * g, t * r ** 3 * inner, 0.0 if dtotal is None else dtotal.double()
    dx = direct - back + past
    # the sum over a row's products is off by its depth times their magnitudes
    off = t.abs() * r ** 3 * (w * g * t).abs().mean(-1, keepdim=True)
    x_bound = BF16 * dx.abs() + 4 * NORM * (direct.abs() + off + (0.0 if dtotal is None else past.abs()))
    terms = g * t * r
    dw = terms.sum(0)
    w_bound = (total.size(0) * 2.0 ** -24 + 2 * NORM) * terms.abs().sum(0) + (BF16 * dw.abs() if weight.dtype == torch.bfloat16 else 0.0)
    return dx, x_bound, dw, w_bound


def select(logits, k, renormalize):
    """(idx, weights in 64 bits): the k largest by a stable sort."""
    values, order = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    values, order = values[:, :k], order[:, :k]
    gone = values == -torch.inf
    over = torch.logsumexp(values if renormalize else logits.double(), -1, keepdim=True)
    return order.masked_fill(gone, -1), torch.where(gone, torch.zeros_like(values), torch.exp(values - over))


def experts(x, idx, weights, w13, w2, s13=None, s2=None, first=0):
    """(out, bound) of the experts of every token.

    The bound follows the kernels: gate and up are sums of H products in fp32, added up in steps of 16 (a step may truncate: a whole ulp); silu' is at most 1.1;
    h is kept to 2^-16 (bf16 weights: two bf16 numbers) or 2^-11 and 2^-24 of the largest of 128 (e4m3 weights); next to e4m3 weights x is exact to 2^-24 of its largest."""
    def wide(w, s, e):
        return w[e].double() if s is None else w[e].double() * s[e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)

    out, bound = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    inter, hidden, fp8 = w2.size(2), w2.size(1), s13 is not None
    for e in range(w13.size(0)):
        t, k = (idx == e + first).nonzero(as_tuple=True)
        if t.numel() == 0 or e + first < 0:
            continue
        rows, a = x[t].double(), wide(w13, s13, e)
        both = rows @ a.T
        slack = (hidden / 16 + 32) * 2.0 ** -23 * (rows.abs() @ a.abs().T)
        if fp8:
            slack = slack + 2.0 ** -24 * rows.abs().amax(-1, keepdim=True) * a.abs().sum(-1)[None]
        g, u, dg, du = both[:, :inter], both[:, inter:], slack[:, :inter], slack[:, inter:]
        act, share = g * torch.sigmoid(g), weights[t, k].double()[:, None]
        h = act * u * share
        dh = (1.1 * dg * u.abs() + (act.abs() + 1.1 * dg) * du) * share.abs() + (2.0 ** -20 + (FP16 if fp8 else 2.0 ** -16)) * h.abs()
        if fp8:
            dh = dh + 2.0 ** -23 * h.abs().amax(-1, keepdim=True)
        b = wide(w2, s2, e)
        out.index_add_(0, t, h @ b.T)
        bound.index_add_(0, t, (dh + (inter / 16 + 64) * 2.0 ** -23 * h.abs()) @ b.abs().T)
    return out, bound + BF16 * (out.abs() + bound)


def quantise(w):
    """e4m3 with one fp32 scale per block of 128 x 128."""
    n, r, c = w.shape
    b = w.float().view(n, r // 128, 128, c // 128, 128)
    s = b.abs().amax(dim=(2, 4)).clamp(min=1e-4) / 448.0
    return (b / s[:, :, None, :, None]).view(n, r, c).to(torch.float8_e4m3fn), s.contiguous()


def layer_inputs(tokens, hidden, inter, local, topk, fp8, device, seed=0, experts_total=None, dropped=0.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    total = experts_total or local
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    w13 = (torch.randn(local, 2 * inter, hidden, generator=g) * 0.05).to(torch.bfloat16)
    w2 = (torch.randn(local, hidden, inter, generator=g) * 0.05).to(torch.bfloat16)
    idx = torch.rand(tokens, total, generator=g).topk(topk, dim=-1).indices
    idx[torch.rand(tokens, topk, generator=g) < dropped] = -1
    weights = torch.softmax(torch.randn(tokens, topk, generator=g), -1)
    s13 = s2 = None
    if fp8:
        (w13, s13), (w2, s2) = quantise(w13), quantise(w2)
    return [None if v is None else v.to(device) for v in (x, idx, weights, w13, w2, s13, s2)]
