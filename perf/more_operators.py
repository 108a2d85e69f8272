"""Performance cases of answering with several hypotheses from the 8-bit cache: what a program that searches with
beams, or serves many sequences that share a prompt, calls beside the decoder's operators.

``listed()`` names fixed cases, ``draw()`` gives others of the same ranges, ``prepare()`` makes what a
program holds before the call, ``run()`` is one pass (elementary torch operations, or the calls of
``axs.unified`` where ``own`` is true), ``work()`` what a pass cannot do without and ``exact()`` the same
result in 64 bits.

Kinds of work:
  select   the best continuations of each sequence's beams over beams and vocabulary
  copy     sequences of the 8-bit cache moved: beams after their parents, a prompt forked, finished ones closed up
  shared   attention of the newest tokens over a prefix that sequences share, and over each one's own cache

Layouts: logits (G, W, V) of W beams for each of G sequences; queries (B, Tq, Hq, D).  The cache holds blocks of
32 tokens: key codes (B, Hkv, blocks, 32, D) and value codes (B, Hkv, blocks, D, 32) in int8, a float32 scale for
each block and head of both, and the raw keys and values of the block that is not yet full, (B, Hkv, 32, D).
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
        # the vocabulary of this repository's example, one sequence with few beams: launches count
        dict(name="select_1x4x256_f32", kind="select", G=1, W=4, V=256, count=4, dtype="f32"),
        # a batch with a large vocabulary in float32; twice as many candidates as beams
        dict(name="select_8x8x32000_f32", kind="select", G=8, W=8, V=32000, count=16, dtype="f32"),
        # an odd vocabulary, rows at any alignment, many beams
        dict(name="select_3x48x50001_f16", kind="select", G=3, W=48, V=50001, count=48, dtype="f16"),
        # a full batch with the largest vocabulary
        dict(name="select_64x8x128000_bf16", kind="select", G=64, W=8, V=128000, count=16, dtype="bf16"),
        # the first steps after a prompt: a handful of tokens a beam
        dict(name="copy_beams_1x4x40", kind="copy", how="beams", G=1, W=4, Hkv=8, D=128, longest=40, capacity=512,
             dtype="bf16"),
        # a batch of beams, each with its own long answer
        dict(name="copy_beams_32x8x2047", kind="copy", how="beams", G=32, W=8, Hkv=8, D=128, longest=2047,
             capacity=2048, dtype="bf16"),
        # prompts' caches forked into eight sequences each, in another cache; heads of 80
        dict(name="copy_fork_8x8x4001", kind="copy", how="fork", G=8, W=8, Hkv=12, D=80, longest=4001, capacity=4096,
             dtype="f16"),
        # a serving batch closes up after a quarter of its sequences ended
        dict(name="copy_close_256x1500", kind="copy", how="close", G=1, W=256, Hkv=4, D=64, longest=1500,
             capacity=2048, dtype="f32"),
        # a short conversation's beams: latency counts
        dict(name="shared_1x4_300_f32", kind="shared", P=1, W=4, Tq=1, Hq=32, Hkv=8, D=128, prefix=300, longest=20,
             capacity=64, dtype="f32"),
        # a batch of long prompts, eight beams each
        dict(name="shared_8x8_16383_bf16", kind="shared", P=8, W=8, Tq=1, Hq=64, Hkv=8, D=128, prefix=16383,
             longest=511, capacity=512, dtype="bf16"),
        # one long system prompt before many conversations
        dict(name="shared_1x128_32000_bf16", kind="shared", P=1, W=128, Tq=1, Hq=32, Hkv=8, D=128, prefix=32000,
             longest=1023, capacity=1024, dtype="bf16"),
        # several new tokens a sequence (drafted ones to be checked), heads of 80, odd lengths
        dict(name="shared_3x21_7777_f16", kind="shared", P=3, W=21, Tq=5, Hq=12, Hkv=4, D=80, prefix=7777,
             longest=333, capacity=352, dtype="f16"),
    ]


def _log(rng, lo, hi) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["select", "copy", "shared"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "select":
        G, W = _log(rng, 1, 64), _log(rng, 1, 64)
        most = 64 * 8 * 128000 // (2 if dtype == "f32" else 1) // (G * W)
        V = _log(rng, 257, max(512, min(160000, most)))
        return dict(kind=kind, G=G, W=W, V=V, count=W * rng.choice([1, 2]), dtype=dtype)
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128])
    if kind == "copy":
        how = rng.choice(["beams", "beams", "fork", "close"])
        G, W = (1, _log(rng, 8, 256)) if how == "close" else (_log(rng, 1, 32), _log(rng, 2, 32))
        longest = _log(rng, 17, max(32, min(16000, (32 * 8 * 2047 * 8 * 128) // (G * W * Hkv * D))))
        return dict(kind=kind, how=how, G=G, W=W, Hkv=Hkv, D=D, longest=longest, capacity=longest + rng.randint(0, 64),
                    dtype=dtype)
    P, W, Tq, g = _log(rng, 1, 16), _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 5]), rng.choice([1, 4, 8])
    # bytes of the sequences' own caches, and (row, key) pairs, of no more than the largest listed case's
    longest = _log(rng, max(2, Tq), max(16, min(1024, (128 * 1023 * 8 * 128) // (P * W * Hkv * D))))
    prefix = _log(rng, 33, max(64, min(65536, (8 * 8 * 64 * 16383 * 128) // (P * W * Tq * g * Hkv * D))))
    return dict(kind=kind, P=P, W=W, Tq=Tq, Hq=Hkv * g, Hkv=Hkv, D=D, prefix=prefix, longest=longest,
                capacity=longest + rng.randint(0, 64), dtype=dtype)


def _lengths(longest: int, n: int, least: int = 1) -> list[int]:
    """Lengths from about a quarter of the longest up to it, the same ones for every seed."""
    return [max(least, longest - (longest * 3 // 4) * b // max(1, n - 1)) for b in range(n)] if n > 1 else [longest]


def _parents(W: int) -> list[int]:
    """Which beam each one continues: half of them go on, the best ones several times."""
    return [i * (i + 1) // (2 * W) for i in range(W)]


def _token_bytes(c: dict, tokens: int) -> int:
    """Bytes of the cache that `tokens` tokens of one sequence take: codes, scales and raw rows of a partial block."""
    blocks = -(-tokens // BLOCK)
    return 2 * c["Hkv"] * (blocks * (BLOCK * c["D"] + 4) + tokens % BLOCK * c["D"] * SIZE[c["dtype"]])


def work(c: dict) -> dict:
    s = SIZE[c["dtype"]]
    if c["kind"] == "select":
        n = c["G"] * c["W"]
        live = n - _finished(c["G"], c["W"])
        return {"bytes": live * c["V"] * s + n * 5 + c["G"] * c["count"] * 20, "flops": 0}
    if c["kind"] == "copy":
        if c["how"] == "beams":
            f = _parents(c["W"])
            moved = [p for i, p in enumerate(f) if p != i]
            return {"bytes": (len(set(moved)) + len(moved)) * sum(_token_bytes(c, n) for n in _lengths(c["longest"], c["G"])),
                    "flops": 0}
        if c["how"] == "fork":
            return {"bytes": (1 + c["W"]) * sum(_token_bytes(c, n) for n in _lengths(c["longest"], c["G"])), "flops": 0}
        live = c["W"] - -(-c["W"] // 4)
        return {"bytes": 2 * sum(_token_bytes(c, n) for n in _lengths(c["longest"], live)), "flops": 0}
    B = c["P"] * c["W"]
    prefix, tails = sum(_lengths(c["prefix"], c["P"])), sum(_lengths(c["longest"], B, c["Tq"]))
    rows = c["Tq"] * c["Hq"] * c["D"]
    nbytes = 2 * (prefix + tails) * c["Hkv"] * (c["D"] + 4 / BLOCK) + 2 * s * B * rows
    return {"bytes": nbytes, "flops": 4 * rows * (prefix * c["W"] + tails)}


# ---- inputs -----------------------------------------------------------------------


def _finished(G: int, W: int) -> int:
    """How many of the beams have ended."""
    return G * W // 10


def _cache(c, B, g, capacity):
    """A cache as quantizing normal values by blocks leaves it."""
    H, D, nb = c["Hkv"], c["D"], -(-capacity // BLOCK)
    codes = [(torch.randn(B, H, nb, *x, generator=g, device="cuda", dtype=torch.float16) * 34).round()
             .clamp(-127, 127).to(torch.int8) for x in ((BLOCK, D), (D, BLOCK))]
    scales = [(torch.rand(B, H, nb, generator=g, device="cuda") + 1) / 45 for _ in range(2)]
    tails = [torch.randn(B, H, BLOCK, D, generator=g, device="cuda").to(DTYPES[c["dtype"]]) for _ in range(2)]
    return (codes[0], scales[0], codes[1], scales[1], tails[0], tails[1])


def prepare(c: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def mixed(values):
        return torch.tensor(values, device="cuda")[torch.randperm(len(values), generator=g, device="cuda")]

    s = {"case": c}
    if c["kind"] == "select":
        G, W, V = c["G"], c["W"], c["V"]
        s["logits"] = (2.5 * torch.randn(G, W, V, generator=g, device="cuda")).to(DTYPES[c["dtype"]])
        # hypotheses of some tokens, within a few units of each other
        s["scores"] = -8 - 4 * torch.rand(G, W, generator=g, device="cuda")
        n = _finished(G, W)
        s["finished"] = mixed([1] * n + [0] * (G * W - n)).bool().view(G, W)
        s["end"] = V // 3
    elif c["kind"] == "copy":
        G, W = c["G"], c["W"]
        if c["how"] == "beams":
            s["cache"] = _cache(c, G * W, g, c["capacity"])
            # the same shape of a family tree for every seed, its members' places mixed
            p = torch.rand(G, W, generator=g, device="cuda").argsort(1)
            f = torch.tensor(_parents(W), device="cuda")
            s["sources"] = torch.empty_like(p).scatter_(1, p, p.gather(1, f.expand(G, W)))
            s["lengths"] = mixed(_lengths(c["longest"], G)).repeat_interleave(W)
        elif c["how"] == "fork":
            s["cache"], s["target"] = _cache(c, G, g, c["capacity"]), _cache(c, G * W, g, c["capacity"])
            s["sources"] = torch.zeros(G, W, device="cuda", dtype=torch.int64)
            s["lengths"] = mixed(_lengths(c["longest"], G))
        else:
            s["cache"] = _cache(c, W, g, c["capacity"])
            # one of every four has ended, the first among them; the others move up, and behind them nothing changes
            off = torch.randint(0, 4, (-(-W // 4),), generator=g, device="cuda")
            off[0] = 0
            ended = (4 * torch.arange(off.numel(), device="cuda") + off).clamp_max(W - 1)
            alive = torch.ones(W, device="cuda", dtype=torch.bool).index_fill_(0, ended, False).nonzero()[:, 0]
            s["sources"] = torch.full((W,), -1, device="cuda", dtype=torch.int64)
            s["sources"][:alive.numel()] = alive
            s["lengths"] = torch.zeros(W, device="cuda", dtype=torch.int64)
            s["lengths"][alive] = mixed(_lengths(c["longest"], alive.numel()))
    else:
        B = c["P"] * c["W"]
        s["q"] = torch.randn(B, c["Tq"], c["Hq"], c["D"], generator=g, device="cuda").to(DTYPES[c["dtype"]])
        s["prefix"], s["cache"] = _cache(c, c["P"], g, c["prefix"]), _cache(c, B, g, c["capacity"])
        s["prefix_lengths"] = mixed(_lengths(c["prefix"], c["P"]))
        s["lengths"] = mixed(_lengths(c["longest"], B, c["Tq"]))
    return s


# ---- one pass ---------------------------------------------------------------------


def run(s: dict):
    c = s["case"]
    if own:
        return _run_own(s, c)
    with torch.no_grad():
        return {"select": _plain_select, "copy": _plain_copy, "shared": _plain_shared}[c["kind"]](s, c)


def _run_own(s, c):
    axu = _axu()
    if c["kind"] == "select":
        return axu.axs_beam_select_unified(s["logits"], s["scores"], s["finished"], s["end"], c["count"])
    if c["kind"] == "copy":
        target = s.get("target")
        axu.axs_cache_copy_unified(axu.AXSKVCacheUnified(*s["cache"]), s["sources"], s["lengths"],
                                   target and axu.AXSKVCacheUnified(*target))
        return target or s["cache"]
    return axu.axs_cache_shared_attention_unified(s["q"], axu.AXSKVCacheUnified(*s["prefix"]), s["prefix_lengths"],
                                                  axu.AXSKVCacheUnified(*s["cache"]), s["lengths"])


def _plain_select(s, c):
    """Log probabilities and their order in 64 bits: in 32, candidates of two beams that lie next to each other
    change places.  Equal ones stand in the order of beams and tokens."""
    G, W, V = c["G"], c["W"], c["V"]
    z = s["logits"].double()
    z -= z.amax(-1, keepdim=True)
    z -= z.exp().sum(-1, keepdim=True).log()
    z += s["scores"].double()[..., None]
    # a beam that has ended goes on as it is
    z.masked_fill_(s["finished"][..., None], -math.inf)
    z[..., s["end"]] = torch.where(s["finished"], s["scores"].double(), z[..., s["end"]])
    top, at = z.view(G, W * V).sort(dim=-1, descending=True, stable=True)
    top, at = top[:, :c["count"]], at[:, :c["count"]]
    none = top == -math.inf   # fewer candidates than asked for
    return top.float(), (at // V).masked_fill_(none, 0), (at % V).masked_fill_(none, 0)


def _plain_copy(s, c):
    """Each of the cache's tensors gathered by source; kept where a sequence has no source or the source no token."""
    cache, target = s["cache"], s.get("target") or s["cache"]
    src, W, B = s["sources"], c["W"], cache[0].shape[0]
    if src.dim() == 2:   # numbers within the group
        src = (src + torch.arange(c["G"], device="cuda")[:, None] * (B // c["G"])).view(-1)
    use, src = src >= 0, src.clamp_min(0)
    n = torch.where(use, s["lengths"][src], 0)
    block = torch.arange(cache[0].shape[2], device="cuda") < (-(-n // BLOCK))[:, None]     # (Bt, blocks)
    row = torch.arange(BLOCK, device="cuda") < (n % BLOCK)[:, None]                        # (Bt, 32)
    for x, y in zip(cache, target):
        keep = row[:, None, :, None] if x.dim() == 4 else block[:, None].view(block.shape[0], 1, -1, *[1] * (x.dim() - 3))
        y.copy_(torch.where(keep, x[src], y))
    return target


def _plain_shared(s, c):
    P, W, Tq, Hq, H, D = (c[x] for x in ("P", "W", "Tq", "Hq", "Hkv", "D"))
    B, g, f = P * W, Hq // H, torch.float32
    off = s["prefix_lengths"].repeat_interleave(W)
    last = (off + s["lengths"])[:, None] - Tq + torch.arange(Tq, device="cuda")   # a query's place, (B, Tq)
    scores, values = [], []
    # the prefix's rows: all queries of the sequences that share it
    for (kc, ks, vc, vs), n, sets, first in ((s["prefix"][:4], s["prefix_lengths"], P, torch.zeros_like(off)),
                                             (s["cache"][:4], s["lengths"], B, off)):
        keys = kc.shape[2] * BLOCK
        k = (kc.to(f) * ks[..., None, None]).view(sets, H, keys, D)
        values.append((vc.to(f) * vs[..., None, None]).transpose(-1, -2).reshape(sets, H, keys, D))
        q = s["q"].to(f).view(sets, B // sets, Tq, H, g, D).permute(0, 3, 1, 2, 4, 5).reshape(sets, H, -1, D)
        x = torch.matmul(q, k.transpose(-1, -2)).mul_(1 / math.sqrt(D)).view(sets, H, B // sets, Tq, g, keys)
        j = torch.arange(keys, device="cuda")
        seen = (j < n.repeat_interleave(B // sets)[:, None, None]) & (j + first[:, None, None] <= last[..., None])
        x.masked_fill_(~seen.view(sets, 1, B // sets, Tq, 1, keys), -math.inf)
        scores.append(x)
    tops = [x.amax(-1, keepdim=True).view(P, H, W, Tq, g, 1) if x.shape[0] == P
            else x.amax(-1, keepdim=True).view(P, W, H, Tq, g, 1).transpose(1, 2) for x in scores]
    top = torch.maximum(*tops).clamp_min(torch.finfo(f).min)
    out, total = 0, 0
    for x, v in zip(scores, values):
        # (sets, H, sequences of a set, Tq, g, 1) of the rows' maxima
        m = top if x.shape[0] == P else top.transpose(1, 2).reshape(B, H, 1, Tq, g, 1)
        x.sub_(m).exp_()
        o = torch.matmul(x.view(x.shape[0], H, -1, x.shape[-1]), v).view(*x.shape[:-1], D)
        l = x.sum(-1, keepdim=True)
        o, l = (y.view(P, H, W, Tq, g, -1) if x.shape[0] == P else y.view(P, W, H, Tq, g, -1).transpose(1, 2)
                for y in (o, l))
        out, total = out + o, total + l
    out = out / total.clamp_min(torch.finfo(f).tiny)
    return out.permute(0, 2, 3, 1, 4, 5).reshape(B, Tq, Hq, D).to(DTYPES[c["dtype"]])


# ---- the definition in 64 bits ------------------------------------------------------


def exact(c: dict, seed: int):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"select": _exact_select, "copy": _exact_copy, "shared": _exact_shared}[c["kind"]](s, c)


def _exact_select(s, c):
    """Sequence by sequence and beam by beam: the best of a beam's own logits in order, then of all beams' best."""
    G, W, V, C = c["G"], c["W"], c["V"], c["count"]
    scores, parents, tokens = [], [], []
    ended = s["finished"].tolist()
    for g in range(G):
        best, at = [], []
        for w in range(W):
            score = s["scores"][g, w].double()
            if ended[g][w]:
                best.append(score[None])
                at.append(torch.tensor([w * V + s["end"]], device="cuda"))
                continue
            z = s["logits"][g, w].double()
            order = z.argsort(dim=-1, descending=True, stable=True)[:C]
            best.append(score + z[order] - torch.logsumexp(z, 0))
            at.append(w * V + order)
        best, at = torch.cat(best), torch.cat(at)
        order = best.argsort(dim=-1, descending=True, stable=True)[:C]
        empty = C - order.numel()
        scores.append(torch.nn.functional.pad(best[order], (0, empty), value=-math.inf))
        parents.append(torch.nn.functional.pad(at[order] // V, (0, empty)))
        tokens.append(torch.nn.functional.pad(at[order] % V, (0, empty)))
    return torch.stack(scores), torch.stack(parents), torch.stack(tokens)


def _exact_copy(s, c):
    """Sequence by sequence: the blocks and raw rows that the source's length reaches."""
    cache = s["cache"]
    out = [x.clone() for x in s.get("target") or cache]
    per = cache[0].shape[0] // c["G"]
    lengths = s["lengths"].tolist()
    for i, p in enumerate(s["sources"].view(-1).tolist()):
        if p < 0:
            continue
        p += i // c["W"] * per if s["sources"].dim() == 2 else 0
        blocks, rows = -(-lengths[p] // BLOCK), lengths[p] % BLOCK
        for k, x in enumerate(cache):
            if k < 4:
                out[k][i, :, :blocks] = x[p, :, :blocks]
            else:
                out[k][i, :, :rows] = x[p, :, :rows]
    return tuple(out[:4]) + tuple(x.double() for x in out[4:])


def _exact_shared(s, c):
    """Prefix by prefix and head by head: softmax(q k^T / sqrt(D)) v over the prefix's values and each sequence's own."""
    P, W, Tq, Hq, H, D = (c[x] for x in ("P", "W", "Tq", "Hq", "Hkv", "D"))
    if work(c)["flops"] > 2e12:
        return None
    g = Hq // H
    out = torch.zeros(P * W, Tq, Hq, D, device="cuda", dtype=torch.float64)

    def values(cache, b, n):
        nb = -(-n // BLOCK)
        k = (cache[0][b, :, :nb].double() * cache[1][b, :, :nb, None, None].double()).flatten(1, 2)
        v = (cache[2][b, :, :nb].double() * cache[3][b, :, :nb, None, None].double()).transpose(2, 3).flatten(1, 2)
        return k[:, :n].contiguous(), v[:, :n].contiguous()

    lengths = s["lengths"].tolist()
    for p, n in enumerate(s["prefix_lengths"].tolist()):
        pk, pv = values(s["prefix"], p, n)
        for b in range(p * W, (p + 1) * W):
            k, v = values(s["cache"], b, lengths[b])
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
            q = s["q"][b].double().view(Tq, H, g, D).permute(1, 0, 2, 3).reshape(H, Tq * g, D)
            x = torch.bmm(q, k.transpose(1, 2).contiguous()).view(H, Tq, g, -1) / math.sqrt(D)
            place = n + lengths[b] - Tq + torch.arange(Tq, device="cuda")
            x.masked_fill_((torch.arange(x.shape[-1], device="cuda") > place[:, None])[:, None], -math.inf)
            y = torch.bmm(torch.softmax(x, -1).view(H, Tq * g, -1), v)
            out[b] = y.view(H, Tq, g, D).permute(1, 0, 2, 3).reshape(Tq, Hq, D)
    return out
