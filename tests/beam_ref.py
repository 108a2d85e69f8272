"""Plain 64-bit forms of beam search's selection, the copying of cached sequences and
attention over a shared prefix."""
from __future__ import annotations

import math

import torch

import decoder_ref as ref


def select(logits, scores, finished=None, end=None, count=None):
    """(scores float64, parents, tokens), each (G, count)."""
    z, c = logits.double().cpu(), scores.double().cpu()
    G, W, V = z.shape
    count = W if count is None else count
    out = torch.full((G, count), -math.inf, dtype=torch.float64)
    parents, tokens = torch.zeros(G, count, dtype=torch.int64), torch.zeros(G, count, dtype=torch.int64)
    for g in range(G):
        s = torch.full((W, V), -math.inf, dtype=torch.float64)
        bad = False
        for w in range(W):
            bad = bad or not bool(c[g, w] < math.inf)
            if finished is not None and bool(finished[g, w]):
                s[w, end] = c[g, w]
            elif c[g, w] != -math.inf:
                top = z[g, w].max()
                bad = bad or not bool(top < math.inf)
                if top > -math.inf:
                    s[w] = c[g, w] + ((z[g, w] - top) - (z[g, w] - top).exp().sum().log())
        if bad:
            out[g] = math.nan
            continue
        best, at = s.view(-1).sort(descending=True, stable=True)
        n = min(count, int((best > -math.inf).sum()))
        out[g, :n], parents[g, :n], tokens[g, :n] = best[:n], at[:n] // V, at[:n] % V
    return out, parents, tokens


def select_bound(want, V):
    """How far a score may be: its rounding to float32, and the logarithm of a sum of float32 exponentials: each is
    off by its own rounding (2 * 2^-24) and by its argument's, 2 * 2^-24 for each unit that it lies below the largest;
    weighted with themselves these are at most log V units."""
    return (want.abs() + 2 * (2 + math.log(V))) * 2.0 ** -24


def copy(cache, sources, lengths, target=None):
    """The target's tensors afterwards, on the CPU."""
    old = [x.cpu() for x in cache]
    out = [x.cpu().clone() for x in (cache if target is None else target)]
    src = sources.cpu().long()
    groups, each = (1, src.numel()) if src.dim() == 1 else src.shape
    per = old[0].shape[0] // groups if groups else 0
    cap = 32 * min(old[0].shape[2], out[0].shape[2])
    for i, p in enumerate(src.reshape(-1).tolist()):
        if not 0 <= p < per:
            continue
        p += i // each * per
        n = min(max(int(lengths[p]), 0), cap)
        for k, x in enumerate(old):
            end = -(-n // 32) if k < 4 else n % 32
            out[k][i, :, :end] = x[p, :, :end]
    return out


def shared_attention(q, prefix, np, own, n, scale=None):
    """q (B, Tq, Hq, D); prefix[p], own[b]: (keys, values) of the tokens that the caches hold, (tokens, H, D) float."""
    B, Tq, Hq, D = q.shape
    W = B // len(prefix)
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64)
    for b in range(B):
        (pk, pv), (k, v) = prefix[b // W], own[b]
        k, v = torch.cat([pk[:np[b // W]], k[:n[b]]]).double(), torch.cat([pv[:np[b // W]], v[:n[b]]]).double()
        T = k.shape[0]
        # queries before the first token see nothing
        mask = (torch.arange(T) <= torch.arange(Tq)[:, None] + (T - Tq))[None, None]
        if T:
            out[b] = ref.attention(q[b:b + 1], k[None], v[None], mask=mask, scale=scale)[0]
    return out
