"""Performance cases of the decoder's operators: what a program that trains a quantized decoder from a
teacher, and then answers with it, calls beside the quantized linear.

``listed()`` names fixed cases, ``draw()`` gives others of the same ranges, ``prepare()`` makes what a
program holds before the call, ``run()`` is one pass (elementary torch operations in 32 bits, or the calls of
``axs.unified`` where ``own`` is true), ``work()`` what a pass cannot do without and ``exact()`` the same
result in 64 bits.

Kinds of work:
  rotary   rotary positions of queries and keys in one call; with ``train`` their gradients too
  attend   attention of grouped heads; with ``train`` the gradients of queries, keys and values
  append   new tokens' keys and values into the 8-bit cache, and the values that the cache then stands for
  decode   attention of the newest tokens over the 8-bit cache
  distill  the distillation loss from a teacher's top logits and its gradient

Layouts: queries (B, T, Hq, D), keys and values (B, T, Hkv, D).  The cache holds blocks of 32 tokens: key
codes (B, Hkv, blocks, 32, D) and value codes (B, Hkv, blocks, D, 32) in int8, a float32 scale for each block
and head of both, and the raw keys and values of the block that is not yet full, (B, Hkv, 32, D).
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32   # tokens of a cache block


def _axu():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "axs-6_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import axs.unified as axu

    return axu


def listed() -> list[dict]:
    return [
        # one new token of a batch of sequences: the smallest call, launches count
        dict(name="rotary_decode_16", kind="rotary", B=16, T=1, Hq=32, Hkv=8, D=128, R=128, interleaved=False,
             positions=8192, dtype="bf16", train=False),
        # a training batch, half of each head rotated in the interleaved layout, forward and backward
        dict(name="rotary_train_4x4095", kind="rotary", B=4, T=4095, Hq=32, Hkv=8, D=128, R=64, interleaved=True,
             positions=4096, dtype="f32", train=True),
        # the small decoder of this repository's training benchmark: batch 64, context 128, 4 heads of 64, float32
        dict(name="attend_train_64x128_f32", kind="attend", B=64, Tq=128, Tk=128, Hq=4, Hkv=4, D=64, causal=True,
             padded=False, dtype="f32", train=True),
        # a training batch of a mid-size decoder with shared key and value heads
        dict(name="attend_train_2x4096_bf16", kind="attend", B=2, Tq=4096, Tk=4096, Hq=32, Hkv=8, D=128, causal=True,
             padded=False, dtype="bf16", train=True),
        # an encoder's batch of sequences of unequal length behind a padding mask, odd sizes
        dict(name="attend_train_pad_777_f16", kind="attend", B=8, Tq=777, Tk=777, Hq=12, Hkv=12, D=80, causal=False,
             padded=True, dtype="f16", train=True),
        # a long prompt, forward alone
        dict(name="attend_prompt_16384_bf16", kind="attend", B=1, Tq=16384, Tk=16384, Hq=16, Hkv=2, D=128,
             causal=True, padded=False, dtype="bf16", train=False),
        # generation: each sequence's one new token into the cache
        dict(name="append_64x1", kind="append", B=64, n=1, Hkv=8, D=128, capacity=4096, dtype="bf16"),
        # a prompt's keys and values into the cache, the last block left partial
        dict(name="append_4x8191", kind="append", B=4, n=8191, Hkv=8, D=128, capacity=8192, dtype="bf16"),
        # one short conversation, one token: latency counts
        dict(name="decode_1x300", kind="decode", B=1, Tq=1, Hq=32, Hkv=8, D=128, longest=300, capacity=512,
             dtype="f32"),
        # a full batch of long conversations of unequal length
        dict(name="decode_64x16384", kind="decode", B=64, Tq=1, Hq=64, Hkv=8, D=128, longest=16383, capacity=16384,
             dtype="bf16"),
        # a small vocabulary in float32
        dict(name="distill_509x1000_f32", kind="distill", N=509, V=1000, K=8, dtype="f32"),
        # a large vocabulary and many tokens in 16 bits
        dict(name="distill_8192x128000_bf16", kind="distill", N=8192, V=128000, K=64, dtype="bf16"),
    ]


def _log(rng, lo, hi) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "attend", "attend", "attend", "append", "decode", "decode", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "rotary":
        Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128])
        Hq = Hkv * rng.choice([1, 3, 4])
        B, R = _log(rng, 1, 16), rng.choice([D, D // 2])
        T = _log(rng, 1, max(1, min(16384, (4 * 4095 * 40 * 128) // (B * (Hq + Hkv) * D))))
        return dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, R=R, interleaved=rng.random() < 0.5,
                    positions=T + rng.randint(0, 4096), dtype=dtype, train=rng.random() < 0.5)
    if kind == "attend":
        Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128])
        Hq, B = Hkv * rng.choice([1, 2, 4]), _log(rng, 1, 16)
        train = rng.random() < 0.6
        most = int(math.sqrt((2.5e11 if dtype == "f32" else 9e11) / (14 if train else 4) / (B * Hq * D)))
        Tk = _log(rng, 17, max(32, min(16384, most)))
        shape = rng.choice(["same", "same", "few", "other"])
        Tq = Tk if shape == "same" else _log(rng, 1, 16) if shape == "few" else _log(rng, 17, Tk)
        return dict(kind=kind, B=B, Tq=Tq, Tk=Tk, Hq=Hq, Hkv=Hkv, D=D, causal=rng.random() < 0.6,
                    padded=rng.random() < 0.3, dtype=dtype, train=train)
    if kind == "append":
        Hkv, D, B = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128]), _log(rng, 1, 64)
        n = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(16000, (4 * 8191 * 8 * 128) // (B * Hkv * D))))
        return dict(kind=kind, B=B, n=n, Hkv=Hkv, D=D, capacity=n + _log(rng, 64, 512), dtype=dtype)
    if kind == "decode":
        Hkv, D, B = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128]), _log(rng, 1, 64)
        longest = _log(rng, 33, max(64, min(131072, (64 * 16384 * 8 * 128) // (B * Hkv * D))))
        return dict(kind=kind, B=B, Tq=rng.choice([1, 1, 1, 2, 5]), Hq=Hkv * rng.choice([1, 4, 8]), Hkv=Hkv, D=D,
                    longest=longest, capacity=longest + rng.randint(0, 64), dtype=dtype)
    N = _log(rng, 1, 8192)
    V = _log(rng, 257, max(512, min(160000, (8192 * 128000 // (2 if dtype == "f32" else 1)) // N)))
    return dict(kind=kind, N=N, V=V, K=rng.choice([1, 8, 20, 64, 200]), dtype=dtype)


def _lengths(longest: int, B: int, least: int) -> list[int]:
    """Lengths from about a quarter of the longest up to it, the same ones for every seed."""
    return [max(least, longest - (longest * 3 // 4) * b // max(1, B - 1)) for b in range(B)] if B > 1 else [longest]


def _keys(c: dict) -> list[int]:
    return _lengths(c["Tk"], c["B"], 1) if c["padded"] else [c["Tk"]] * c["B"]


def _pairs(c: dict) -> int:
    """(query, key) pairs that attend, of all sequences and one head."""
    total = 0
    for keys in _keys(c):
        if not c["causal"]:
            total += c["Tq"] * keys
            continue
        off = c["Tk"] - c["Tq"]   # query i sees keys up to i + off
        lo, hi = max(0, -off), c["Tq"]
        full = max(lo, min(hi, keys - 1 - off))   # from here on a query sees every key
        total += sum(i + off + 1 for i in range(lo, full)) + (hi - full) * keys
    return total


def work(c: dict) -> dict:
    s = SIZE[c["dtype"]]
    if c["kind"] == "rotary":
        n = c["B"] * c["T"] * (c["Hq"] + c["Hkv"]) * c["D"]
        return {"bytes": (2 if c["train"] else 1) * (2 * n * s + c["B"] * c["T"] * (8 + 4 * c["R"])), "flops": 0}
    if c["kind"] == "attend":
        q, kv = c["B"] * c["Tq"] * c["Hq"] * c["D"], 2 * c["B"] * c["Tk"] * c["Hkv"] * c["D"]
        nbytes = s * (2 * q + kv) + (c["B"] * c["Tk"] if c["padded"] else 0)
        if c["train"]:
            nbytes += s * (2 * q + kv)   # the output's gradient in, the three gradients out
        return {"bytes": nbytes, "flops": (14 if c["train"] else 4) * _pairs(c) * c["Hq"] * c["D"]}
    if c["kind"] == "append":
        n = 2 * c["B"] * c["n"] * c["Hkv"] * c["D"]
        read = 2 * c["B"] * -(-c["n"] // BLOCK) * BLOCK * c["Hkv"] * c["D"]
        # values in, codes out, the partial block raw; then the codes in and what they stand for out
        tail = 2 * c["B"] * c["Hkv"] * c["D"] * (16 if c["n"] == 1 else c["n"] % BLOCK)
        return {"bytes": n * s + read + tail * s + 5 * read, "flops": 0}
    if c["kind"] == "decode":
        keys = sum(_lengths(c["longest"], c["B"], c["Tq"]))
        nbytes = 2 * keys * c["Hkv"] * (c["D"] + 4 / BLOCK) + 2 * s * c["B"] * c["Tq"] * c["Hq"] * c["D"]
        return {"bytes": nbytes, "flops": 4 * keys * c["Tq"] * c["Hq"] * c["D"]}
    return {"bytes": 2 * c["N"] * c["V"] * s + c["N"] * c["K"] * 12, "flops": 0}


# ---- inputs -----------------------------------------------------------------------


def prepare(c: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": c}
    if c["kind"] == "rotary":
        B, T, D, R = c["B"], c["T"], c["D"], c["R"]
        s["q"], s["k"] = randn(B, T, c["Hq"], D), randn(B, T, c["Hkv"], D)
        inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        angle = torch.arange(c["positions"], device="cuda", dtype=torch.float64)[:, None] * inv
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        first = torch.randint(0, c["positions"] - T + 1, (B, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(T, device="cuda")
        if c["train"]:
            s["gq"], s["gk"] = randn(B, T, c["Hq"], D), randn(B, T, c["Hkv"], D)
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
    elif c["kind"] == "attend":
        B, Tq, Tk, D = c["B"], c["Tq"], c["Tk"], c["D"]
        s["q"], s["k"], s["v"] = randn(B, Tq, c["Hq"], D), randn(B, Tk, c["Hkv"], D), randn(B, Tk, c["Hkv"], D)
        if c["padded"]:
            lens = torch.tensor(_keys(c), device="cuda")[torch.randperm(B, generator=g, device="cuda")]
            s["mask"] = (torch.arange(Tk, device="cuda") < lens[:, None])[:, None, None, :].contiguous()
        if c["train"]:
            s["go"] = randn(B, Tq, c["Hq"], D)
            for x in ("q", "k", "v"):
                s[x].requires_grad_(True)
    elif c["kind"] in ("append", "decode"):
        B, H, D, nb = c["B"], c["Hkv"], c["D"], -(-c["capacity"] // BLOCK)
        if c["kind"] == "append":
            s["k"], s["v"] = randn(B, c["n"], H, D), randn(B, c["n"], H, D)
            if c["n"] == 1:   # anywhere in the cache, after tokens of which the last block's are held raw
                s["starts"] = torch.randint(0, c["capacity"], (B,), generator=g, device="cuda")
                tails = randn(B, H, BLOCK, D), randn(B, H, BLOCK, D)
            else:
                s["starts"] = torch.zeros(B, device="cuda", dtype=torch.int64)
                tails = tuple(torch.zeros(B, H, BLOCK, D, device="cuda", dtype=dt) for _ in range(2))
            codes = [torch.zeros(B, H, nb, BLOCK, D, device="cuda", dtype=torch.int8),
                     torch.zeros(B, H, nb, D, BLOCK, device="cuda", dtype=torch.int8)]
            scales = [torch.zeros(B, H, nb, device="cuda") for _ in range(2)]
        else:
            s["q"] = randn(B, c["Tq"], c["Hq"], D)
            lens = torch.tensor(_lengths(c["longest"], B, c["Tq"]), device="cuda")
            s["lengths"] = lens[torch.randperm(B, generator=g, device="cuda")]
            # codes as quantizing normal values by blocks gives them
            codes = [(torch.randn(B, H, nb, *x, generator=g, device="cuda", dtype=torch.float16) * 34).round()
                     .clamp(-127, 127).to(torch.int8) for x in ((BLOCK, D), (D, BLOCK))]
            scales = [(torch.rand(B, H, nb, generator=g, device="cuda") + 1) / 45 for _ in range(2)]
            tails = randn(B, H, BLOCK, D), randn(B, H, BLOCK, D)   # not read
        s["cache"] = (codes[0], scales[0], codes[1], scales[1], tails[0], tails[1])
    else:
        N, V, K = c["N"], c["V"], c["K"]
        s["logits"] = (2 * randn(N, V, dtype=dt)).requires_grad_(True)
        s["values"] = 4 + 2 * randn(N, K, dtype=torch.float32)
        # K different classes of each row: a random start and a random odd step over a power of two
        span = 1 << (V.bit_length() - 1)
        start = torch.randint(0, span, (N, 1), generator=g, device="cuda")
        step = 2 * torch.randint(0, max(1, span // 2), (N, 1), generator=g, device="cuda") + 1
        s["indices"] = (start + step * torch.arange(K, device="cuda")) % span
        s["weights"] = (torch.rand(N, generator=g, device="cuda") < 0.9).float()
        s["weights"][0] = 1.0   # at least one row counts
    return s


# ---- one pass ---------------------------------------------------------------------


def run(s: dict):
    c = s["case"]
    if own:
        return _run_own(s, c)
    with torch.no_grad():
        return _plain(s, c, torch.float32)


def _run_own(s, c):
    axu = _axu()
    if c["kind"] == "rotary":
        if not c["train"]:
            return axu.axs_rotary_unified(s["q"], s["k"], s["table"], s["positions"], c["interleaved"])
        q, k = axu.axs_rotary_unified(s["q"], s["k"], s["table"], s["positions"], c["interleaved"])
        return q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    if c["kind"] == "attend":
        out = axu.axs_attention_unified(s["q"], s["k"], s["v"], s.get("mask"), c["causal"])
        if not c["train"]:
            return out
        return out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["go"])
    if c["kind"] == "append":
        cache = axu.AXSKVCacheUnified(*s["cache"])
        axu.axs_cache_append_unified(cache, s["k"], s["v"], s["starts"])
        first = s["starts"] // BLOCK * BLOCK if c["n"] == 1 else s["starts"]
        values = axu.axs_cache_read_unified(cache, first, -(-c["n"] // BLOCK) * BLOCK)
        return (*values, cache.k_tail, cache.v_tail)
    if c["kind"] == "decode":
        return axu.axs_cache_attention_unified(s["q"], axu.AXSKVCacheUnified(*s["cache"]), s["lengths"])
    loss = axu.axs_distillation_loss_unified(s["logits"], s["values"], s["indices"], 2.0, s["weights"])
    return loss.detach(), *torch.autograd.grad(loss, s["logits"])


def _plain(s, c, f):
    """The operators from elementary operations in the type f; results in the types the calls return."""
    dt = DTYPES[c["dtype"]] if f == torch.float32 else f
    if c["kind"] == "rotary":
        cos, sin = s["table"].to(f)[s["positions"]][:, :, None].chunk(2, -1)
        outs = [_rotate(x.to(f), cos, sin, c).to(dt) for x in (s["q"], s["k"])]
        if c["train"]:
            outs += [_rotate(x.to(f), cos, -sin, c).to(dt) for x in (s["gq"], s["gk"])]
        return tuple(outs)
    if c["kind"] == "attend":
        return _plain_attend(s, c, f, dt)
    if c["kind"] == "append":
        return _plain_append(s, c, f)
    if c["kind"] == "decode":
        return _plain_decode(s, c, f, dt)
    T, w = 2.0, s["weights"].to(f)
    z, t = s["logits"].to(f) / T, s["values"].to(f) / T
    logq = z - z.amax(-1, keepdim=True)
    logq -= logq.exp().sum(-1, keepdim=True).log()
    logp = t - t.amax(-1, keepdim=True)
    logp = logp - logp.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    rows = T * T * (p * (logp - logq.gather(1, s["indices"]))).sum(-1)
    loss = (w * rows).sum() / w.sum()
    grad = logq.exp_()
    grad.scatter_add_(1, s["indices"], -p)
    grad *= (T * w / w.sum())[:, None]
    return loss, grad.to(dt)


def _rotate(x, cos, sin, c):
    R = c["R"]
    y = x.clone()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if c["interleaved"] else (x[..., :R // 2], x[..., R // 2:R])
    if c["interleaved"]:
        y[..., 0:R:2], y[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
    else:
        y[..., :R // 2], y[..., R // 2:R] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_attend(s, c, f, dt):
    B, Tq, Tk, Hq, H, D = (c[x] for x in ("B", "Tq", "Tk", "Hq", "Hkv", "D"))
    g, scale = Hq // H, 1 / math.sqrt(D)

    def queries(x):   # (B, Hkv, g * Tq, D)
        return x.detach().to(f).reshape(B, Tq, H, g, D).permute(0, 2, 3, 1, 4).reshape(B, H, g * Tq, D)

    def heads(x):     # (B, T, H, D) of what queries() or keys() gave
        return x.reshape(B, H, g, Tq, D).permute(0, 3, 1, 2, 4).reshape(B, Tq, Hq, D).to(dt)

    q, k, v = queries(s["q"]), s["k"].detach().to(f).transpose(1, 2), s["v"].detach().to(f).transpose(1, 2)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(B, H, g, Tq, Tk)
    if c["causal"]:
        i, j = torch.arange(Tq, device="cuda")[:, None], torch.arange(Tk, device="cuda")
        p.masked_fill_(j > i + (Tk - Tq), -math.inf)
    if "mask" in s:
        p.masked_fill_(~s["mask"][:, :, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min(torch.finfo(f).min)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min(torch.finfo(f).tiny))
    p = p.view(B, H, g * Tq, Tk)
    out = torch.matmul(p, v)
    if not c["train"]:
        return heads(out)
    go = queries(s["go"])
    dv = torch.matmul(p.transpose(-1, -2), go)
    ds = torch.matmul(go, v.transpose(-1, -2)).sub_((go * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    return heads(out), heads(dq), dk.transpose(1, 2).contiguous().to(dt), dv.transpose(1, 2).contiguous().to(dt)


def _plain_append(s, c, f):
    """The blocks from the one that holds the first new token: the raw values (those of the partial block before
    it from the tail), a scale and codes for each block, and the values that these stand for."""
    B, n, H, D = c["B"], c["n"], c["Hkv"], c["D"]
    at = s["starts"] % BLOCK                                    # the first new token's place in its block
    nb = -(-n // BLOCK)
    place = torch.arange(nb * BLOCK, device="cuda")[None, :]    # places from that block's first
    new = (place >= at[:, None]) & (place < at[:, None] + n)
    values, tails = [], []
    for x, tail in ((s["k"], s["cache"][4]), (s["v"], s["cache"][5])):
        idx = (place - at[:, None]).clamp(0, n - 1)[:, :, None, None].expand(B, -1, H, D)
        raw = torch.where(new[:, :, None, None], x.gather(1, idx), 0)
        old = (place[:, :BLOCK] < at[:, None])[:, :, None, None]
        raw[:, :BLOCK] = torch.where(old, tail.transpose(1, 2), raw[:, :BLOCK])
        blocks = raw.float().view(B, nb, BLOCK, H, D)
        scale = blocks.abs().amax((2, 4), keepdim=True)
        scale = scale / torch.full_like(scale, 127)   # a true division: by a number it would be a product
        codes = (blocks.to(f) / torch.where(scale > 0, scale, 1).to(f)).round().clamp(-127, 127)
        values.append((codes.float() * scale).view(B, nb * BLOCK, H, D))
        # the last block's raw values, kept while it is partial
        last = raw[:, -BLOCK:].transpose(1, 2)
        kept = (new[:, -BLOCK:] & ((at + n) % BLOCK != 0)[:, None])[:, None, :, None]
        tails.append(torch.where(kept, last, tail))
    return (*values, *tails)


def _plain_decode(s, c, f, dt):
    B, Tq, Hq, H, D = (c[x] for x in ("B", "Tq", "Hq", "Hkv", "D"))
    g = Hq // H
    kc, ks, vc, vs = s["cache"][:4]
    nb = kc.shape[2]
    k = (kc.to(f) * ks[..., None, None].to(f)).view(B, H, nb * BLOCK, D)
    q = s["q"].to(f).reshape(B, Tq, H, g, D).permute(0, 2, 3, 1, 4).reshape(B, H, g * Tq, D)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(D)).view(B, H, g, Tq, nb * BLOCK)
    last = s["lengths"][:, None] - Tq + torch.arange(Tq, device="cuda")   # a query's own place
    p.masked_fill_((torch.arange(nb * BLOCK, device="cuda") > last[..., None])[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    del k
    v = (vc.to(f) * vs[..., None, None].to(f)).transpose(-1, -2).reshape(B, H, nb * BLOCK, D)
    out = torch.matmul(p.view(B, H, g * Tq, nb * BLOCK), v).view(B, H, g, Tq, D)
    return out.permute(0, 3, 1, 2, 4).reshape(B, Tq, Hq, D).to(dt)


# ---- the definition in 64 bits ------------------------------------------------------


def exact(c: dict, seed: int):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "attend": _exact_attend, "append": _exact_append, "decode": _exact_decode,
                "distill": _exact_distill}[c["kind"]](s, c)


def _exact_rotary(s, c):
    """Each pair as a complex number times (cos + i sin), or its conjugate for the gradients."""
    R = c["R"]
    tab = s["table"].double()[s["positions"]]
    turn = torch.complex(tab[..., :R // 2], tab[..., R // 2:])[:, :, None]

    def turned(x, by):
        x = x.detach().double()
        pair = x[..., :R].unflatten(-1, (-1, 2) if c["interleaved"] else (2, -1))
        if not c["interleaved"]:
            pair = pair.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * by)
        if not c["interleaved"]:
            y = y.transpose(-1, -2)
        return torch.cat([y.flatten(-2), x[..., R:]], -1)

    outs = [turned(s["q"], turn), turned(s["k"], turn)]
    if c["train"]:
        outs += [turned(s["gq"], turn.conj()), turned(s["gk"], turn.conj())]
    return tuple(outs)


def _exact_attend(s, c):
    """Head by head and some queries at a time: softmax(q k^T / sqrt(D)) v over the keys a query sees."""
    B, Tq, Tk, Hq, D = (c[x] for x in ("B", "Tq", "Tk", "Hq", "D"))
    if _pairs(c) * Hq * D > 4e11:
        return None
    g, off, step = Hq // c["Hkv"], Tk - Tq, 2048
    q, k, v = (s[x].detach().double() for x in ("q", "k", "v"))
    go = s["go"].double() if c["train"] else None
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    j = torch.arange(Tk, device="cuda")
    for b in range(B):
        seen_b = s["mask"][b, 0, 0] if "mask" in s else torch.ones(Tk, device="cuda", dtype=torch.bool)
        for h in range(Hq):
            kh, vh = k[b, :, h // g], v[b, :, h // g]
            for i0 in range(0, Tq, step):
                qi = q[b, i0:i0 + step, h]
                seen = seen_b.expand(qi.shape[0], Tk)
                if c["causal"]:
                    seen = seen & (j <= torch.arange(i0, i0 + qi.shape[0], device="cuda")[:, None] + off)
                x = (qi @ kh.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
                lse = torch.logsumexp(x, -1, keepdim=True)
                p = torch.where(seen, (x - lse).exp(), 0)
                out[b, i0:i0 + step, h] = p @ vh
                if c["train"]:
                    gi = go[b, i0:i0 + step, h]
                    dp = gi @ vh.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[b, i0:i0 + step, h] = ds @ kh
                    dk[b, :, h // g] += ds.T @ qi
                    dv[b, :, h // g] += p.T @ gi
    return (out, dq, dk, dv) if c["train"] else out


def _exact_append(s, c):
    """Sequence by sequence: a block's scale is its largest magnitude over 127, rounded to float32, its codes the
    float32 quotients by it, rounded to even whole numbers; the tails are copies."""
    B, n, D = c["B"], c["n"], c["D"]
    nb = -(-n // BLOCK)
    outs, tails = [], []
    starts = s["starts"].tolist()
    for x, tail in ((s["k"], s["cache"][4]), (s["v"], s["cache"][5])):
        rows, new_tail = [], tail.clone()
        for b in range(B):
            at = starts[b] % BLOCK
            raw = torch.cat([tail[b, :, :at].transpose(0, 1), x[b]], 0)
            end = raw.shape[0]
            raw = torch.nn.functional.pad(raw, (0, 0, 0, 0, 0, nb * BLOCK - end)).double()
            blk = raw.view(nb, BLOCK, -1, D)
            scale = (blk.abs().amax((1, 3), keepdim=True) / 127).float().double()
            codes = torch.where(scale > 0, blk / scale, 0).float().round().double()
            rows.append((codes * scale).view(nb * BLOCK, -1, D))
            if end % BLOCK:
                first = max(0, (nb - 1) * BLOCK - at)   # the new tokens of the last block
                to = 0 if n > 1 else at
                new_tail[b, :, to:end % BLOCK] = x[b, first:].transpose(0, 1)
        outs.append(torch.stack(rows))
        tails.append(new_tail.double())
    return (*outs, *tails)


def _exact_decode(s, c):
    B, Tq, Hq, H, D = (c[x] for x in ("B", "Tq", "Hq", "Hkv", "D"))
    kc, ks, vc, vs = s["cache"][:4]
    out = torch.zeros(B, Tq, Hq, D, device="cuda", dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        nb = -(-n // BLOCK)
        k = (kc[b, :, :nb].double() * ks[b, :, :nb, None, None].double()).flatten(1, 2)
        v = (vc[b, :, :nb].double() * vs[b, :, :nb, None, None].double()).transpose(2, 3).flatten(1, 2)
        for t in range(Tq):
            m = n - Tq + t + 1
            q = s["q"][b, t].double().view(H, Hq // H, D)
            x = torch.bmm(q, k[:, :m].transpose(1, 2)) / math.sqrt(D)
            out[b, t] = torch.bmm(torch.softmax(x, -1), v[:, :m]).reshape(Hq, D)
    return out


def _exact_distill(s, c):
    T, n = 2.0, c["N"]
    w = s["weights"].double()
    loss, grad = 0.0, torch.empty(n, c["V"], device="cuda", dtype=torch.float64)
    for i in range(0, n, 512):
        z = s["logits"][i:i + 512].detach().double() / T
        p = torch.softmax(s["values"][i:i + 512].double() / T, -1)
        idx, wi = s["indices"][i:i + 512], w[i:i + 512, None] / w.sum()
        logq = torch.log_softmax(z, -1)
        loss = loss + (T * T * wi * p * (p.log() - logq.gather(1, idx))).sum()
        grad[i:i + 512] = T * wi * logq.exp().scatter_add(1, idx, -p)
    return loss, grad
