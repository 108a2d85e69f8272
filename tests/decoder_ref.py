"""Plain 64-bit forms of the decoder's operators (rotary positions, attention,
the 8-bit cache, distillation) and the error bounds their tests use.

Bounds follow from the types before any run: u is a type's unit roundoff
(bfloat16 2^-8, float16 2^-11, float32 2^-24).
"""
from __future__ import annotations

import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def rel(got: torch.Tensor, want: torch.Tensor) -> float:
    """2-norm of the difference over that of the result (of the difference where that is 0)."""
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), "NaN in other places"
    d = float((got - want).nan_to_num().norm())
    n = float(want.nan_to_num().norm())
    return d / n if n else d


def rotate(x, table, positions, interleaved, inverse=False):
    """x (B, T, H, D) in 64 bits."""
    x, R = x.double().cpu(), table.shape[1]
    tab = table.double().cpu()[positions.cpu()]
    c, s = tab[..., :R // 2], tab[..., R // 2:]
    if tab.dim() == 2:
        c, s = c[None], s[None]
    c, s = c[:, :, None], (-s if inverse else s)[:, :, None]
    y = x.clone()
    i = torch.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def seen(B, Hq, Tq, Tk, causal, mask):
    """(seen, added): which keys a query sees and what the mask adds, (B, Hq, Tq, Tk)."""
    ok = torch.ones(B, Hq, Tq, Tk, dtype=torch.bool)
    add = torch.zeros(B, Hq, Tq, Tk, dtype=torch.float64)
    if causal:
        ok &= torch.arange(Tk) <= torch.arange(Tq)[:, None] + (Tk - Tq)
    if mask is not None and mask.dtype == torch.bool:
        ok &= mask.cpu()
    elif mask is not None:
        add = add + mask.double().cpu()
        ok &= add != -math.inf
    return ok, add


def seen_product(w, m, x):
    """w x over the pairs of m alone: a weight of 0 elsewhere would turn an infinity or NaN of x into NaN."""
    if x.isfinite().all():
        return w @ x
    return torch.where(m[:, :, None], w[:, :, None] * x[None], 0.0).sum(1)


def attention(q, k, v, go=None, mask=None, causal=False, scale=None):
    """out, or (out, dq, dk, dv) for the output's gradient go; unseen keys have no part in a row."""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    B, Tq, Hq, D = q.shape
    Tk, H = k.shape[1], k.shape[2]
    g = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    ok, add = seen(B, Hq, Tq, Tk, causal, mask)
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        for h in range(Hq):
            kh, vh, qh = k[b, :, h // g], v[b, :, h // g], q[b, :, h]
            m = ok[b, h]
            x = torch.where(m, (qh @ kh.T) * scale + add[b, h], -math.inf)
            top = x.amax(-1, keepdim=True) if Tk else x.new_zeros(Tq, 1)
            e = torch.where(m, (x - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            total = e.sum(-1, keepdim=True)
            p = torch.where(total == 0, 0.0, e / total) if Tk else e   # a NaN total stays
            out[b, :, h] = seen_product(p, m, vh)
            if go is not None:
                gh = go[b, :, h].detach().double().cpu()
                dp = gh @ vh.T
                pdp = torch.where(m, p * dp, 0.0)
                ds = torch.where(m, (pdp - p * pdp.sum(-1, keepdim=True)) * scale, 0.0)
                dq[b, :, h] = seen_product(ds, m, kh)
                dk[b, :, h // g] += seen_product(ds.T, m.T, qh)
                dv[b, :, h // g] += seen_product(p.T, m.T, gh)
    return out if go is None else (out, dq, dk, dv)


def quantize_tokens(x):
    """x (n, H, D) from a block's first token on: codes (n, H, D) and scales (blocks, H), in the cache's arithmetic."""
    n, H, D = x.shape
    nb = -(-n // 32)
    blocks = torch.zeros(nb * 32, H, D)
    blocks[:n] = x.float().cpu()
    blocks = blocks.view(nb, 32, H, D)
    scale = blocks.abs().amax((1, 3)) / torch.tensor(127.0)
    scale = torch.where(blocks.isfinite().all(3).all(1), scale, torch.nan)
    s = scale[:, None, :, None]
    codes = torch.where(s > 0, blocks / s, 0.0).round().clamp(-127, 127).to(torch.int8)
    return codes.view(nb * 32, H, D)[:n], scale


def cache_values(x):
    """The values that tokens x (n, H, D), from a block's first on, have in the cache."""
    codes, scale = quantize_tokens(x)
    return codes.float() * scale.repeat_interleave(32, 0)[:x.shape[0], :, None]


def distill(z, values, indices, T, w=None, reduction="mean"):
    """(loss or rows, gradient of the sum of what comes back) in 64 bits."""
    V, K = z.shape[-1], values.shape[-1]
    z, t = z.detach().double().cpu().reshape(-1, V) / T, values.double().cpu().reshape(-1, K) / T
    idx = indices.cpu().long().reshape(-1, K)
    w = torch.ones(z.shape[0], dtype=torch.float64) if w is None else w.double().cpu().reshape(-1)
    rows, grad = torch.zeros(z.shape[0], dtype=torch.float64), torch.zeros_like(z)
    for r in range(z.shape[0]):
        use = idx[r] >= 0
        if w[r] == 0 or not use.any():
            continue
        if (idx[r] >= V).any():
            rows[r], grad[r] = math.nan, math.nan
            continue
        logp = torch.log_softmax(t[r][use], 0)
        p, logq = logp.exp(), torch.log_softmax(z[r], 0)
        rows[r] = T * T * torch.where(p > 0, p * (logp - logq[idx[r][use]]), 0.0).sum()
        grad[r] = T * (logq.exp() - torch.zeros_like(logq).index_add_(0, idx[r][use], p))
    f = 1.0 / w.sum() if reduction == "mean" and w.sum() != 0 else 0.0 if reduction == "mean" else 1.0
    grad = grad * w[:, None] * f
    rows = torch.where(w == 0, 0.0, rows * w)
    return (rows if reduction == "none" else rows.sum() * f), grad
