"""Beam search's operators on the GPU where single digits, orders or places count: peaked rows, large scores, value
scales far apart, caches past 32 bits, what a search leaves in its caches."""
from __future__ import annotations

import math

import pytest
import torch

import beam_ref
import decoder_ref as ref
from test_gpu_beams import _bound, _check_select, _filled, _gen, _Reader

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("V", [512, 4097, 50001])
def test_peaked_rows_keep_their_order(V, dtype):
    """Each beam's best token is all but certain, and the beams' scores for it lie 2e-8 apart.  A row's sum is then 1
    and a rest r < 4e-3, in which each exponential is off by at most (2 + d) 2^-24 of itself, d the units that it lies below
    the largest, less than 30 for all that count: log(1 + r) is off by 32 r 2^-24 < 8e-9, as long as the sum keeps more digits
    than its terms."""
    W, gap = 16, 2e-8
    g = _gen(V)
    logits = 2 * torch.randn(3, W, V, generator=g)
    peak = torch.randint(0, V, (3, W, 1), generator=g)
    logits = logits.scatter(2, peak, logits.amax(2, keepdim=True) + 11).to(dtype)
    z = logits.double()
    total = (z - z.amax(2, keepdim=True)).exp().sum(2).log()
    assert (total < 4e-3).all()
    place = torch.stack([torch.randperm(W, generator=g) for _ in range(3)])
    scores = (total - 0.01 - gap * place).float()            # of about 0.01: steps of 1e-9
    best = (scores.double() - total).sort(1, descending=True)
    assert (best.values[:, :-1] - best.values[:, 1:] > 0.8 * gap).all() and torch.equal(best.indices, place.argsort(1))
    _check_select(logits.to(DEV), scores.to(DEV), count=W)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_vocabulary(dtype):
    """One row of 2^31 - 1 tokens: its last ones, and more equal ones there than are listed."""
    from axs.unified import axs_beam_select_unified

    V = 2 ** 31 - 1
    logits = torch.full((1, 1, V), -math.inf, device=DEV, dtype=dtype)
    zero = torch.zeros(1, 1, device=DEV)
    at = [V - 1, 0, V - 8, V - 2049, 1 << 30]
    logits[0, 0, at] = torch.tensor([5.0, 4.0, 3.0, 2.0, 1.0], device=DEV, dtype=dtype)
    total = math.log(sum(math.exp(x) for x in range(1, 6)))
    got = axs_beam_select_unified(logits, zero, count=6)
    assert got[2].tolist() == [at + [0]] and not got[1].any()
    want = torch.tensor([[5.0, 4, 3, 2, 1, math.inf]]).double() - total
    want[0, 5] = -math.inf
    assert got[0][0, 5] == -math.inf
    assert ((got[0].cpu() - want)[:, :5].abs() <= beam_ref.select_bound(want, 5)[:, :5]).all()
    logits[0, 0, -700:] = 6
    got = axs_beam_select_unified(logits, zero, count=128)
    assert torch.equal(got[2][0].cpu(), torch.arange(V - 700, V - 572))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_search_under_another_default_dtype(dtype):
    from axs.unified import axs_beam_search_unified

    m, other = _Reader(2, 3, 40, 0, 5), _Reader(2, 3, 40, 0, 5)
    want = axs_beam_search_unified(m, m.logits(m.prompt), m.caches, 3, 6)
    torch.set_default_dtype(dtype)
    try:
        got = axs_beam_search_unified(other, other.logits(other.prompt), other.caches, 3, 6)
    finally:
        torch.set_default_dtype(torch.float32)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("G,W,V,steps,starts", [(1, 4, 60, 2, 0), (3, 5, 90, 33, 0), (2, 3, 50, 20, 29)])
def test_search_leaves_its_beams_in_the_caches(G, W, V, steps, starts):
    """Each sequence of the caches ends as its returned beam: the prompt and all tokens but the last."""
    from axs.unified import axs_beam_search_unified, axs_cache_read_unified

    m = _Reader(G, W, V, starts, 7 + V)
    start = torch.full((G * W,), starts, device=DEV)
    scores, tokens = axs_beam_search_unified(m, m.logits(m.prompt), m.caches, W, steps, None, start)
    assert scores.isfinite().all()
    want = torch.cat([m.prompt.repeat_interleave(W, 0), tokens.cpu().view(G * W, steps)[:, :-1]], 1)
    for c in m.caches:
        k, _ = axs_cache_read_unified(c, torch.zeros_like(start), starts + steps - 1)
        assert torch.equal(k[..., -1, 3].round().long().cpu(), want)


def test_search_of_no_prompts():
    from axs.unified import AXSKVCacheUnified, axs_beam_search_unified

    cache = AXSKVCacheUnified.empty(0, 2, 16, 40, torch.float32, DEV)
    scores, tokens = axs_beam_search_unified(lambda t, s: torch.zeros(0, 1, 9, device=DEV), torch.zeros(0, 9, device=DEV), [cache], 3, 5, 4)
    assert scores.shape == (0, 3) and tokens.shape == (0, 3, 5)


# ---- attention over a shared prefix ------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("W", [2, 40])
def test_shared_values_of_the_largest_size_where_they_are_not_seen(W, dtype):
    """Later tokens of nearly the type's largest size, in the prefix and among a sequence's own: queries before them
    keep theirs, of 1e-3, to the last digit."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_shared_attention_unified

    def filled(B, n, first, seed):
        g = _gen(seed)
        k, v = (torch.randn(B, n, 1, 64, generator=g).to(DEV, dtype) for _ in range(2))
        v *= 1e-3
        v[:, first:] = 0.9 * torch.finfo(dtype).min
        c = AXSKVCacheUnified.empty(B, 1, 64, n, dtype, DEV)
        axs_cache_append_unified(c, k, v, torch.zeros(B, dtype=torch.int64, device=DEV))
        return c, [(ref.cache_values(x), ref.cache_values(y)) for x, y in zip(k, v)]

    q = torch.randn(W, 40, 2, 64, generator=_gen(3)).to(DEV, dtype)
    # own tokens from 32 on: of 60, the last 40 are the queries (two blocks are one workgroup's)
    (prefix, pv), (cache, ov) = filled(1, 64, 64, 1), filled(W, 60, 32, 2)
    call = axs_cache_shared_attention_unified
    out = call(q, prefix, torch.tensor([64], device=DEV), cache, torch.full((W,), 60, device=DEV))
    want = beam_ref.shared_attention(q, pv, [64], ov, [60] * W)
    assert ref.rel(out[:, :12], want[:, :12]) <= _bound(dtype)
    assert ref.rel(out[:, 12:].double() / 2e38, want[:, 12:] / 2e38) <= _bound(dtype)
    # the prefix's from 32 on: of 64 + 1 tokens the last 40 are the queries, the first seven of which stand before them
    (prefix, pv), (cache, ov) = filled(1, 64, 32, 4), filled(W, 1, 1, 5)
    out = call(q, prefix, torch.tensor([64], device=DEV), cache, torch.full((W,), 1, device=DEV))
    want = beam_ref.shared_attention(q, pv, [64], ov, [1] * W)
    assert ref.rel(out[:, :7], want[:, :7]) <= _bound(dtype)
    assert ref.rel(out[:, 7:].double() / 2e38, want[:, 7:] / 2e38) <= _bound(dtype)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("D", [64, 192])
@pytest.mark.parametrize("W", [2, 40])
@pytest.mark.parametrize("size", [64.0, 4000.0, 40000.0, 1e6])
def test_shared_large_scores(W, size, D, dtype):
    """Queries of up to `size` along one key each, whose score passes all others by so much that its value alone
    counts: the output is that value, whatever the score's own size and rounding."""
    from axs.unified import axs_cache_shared_attention_unified

    if size > torch.finfo(dtype).max:
        return
    g = _gen(int(size) + W)
    prefix, pv = _filled(1, 200, 2, D, dtype, 200, 21)
    cache, ov = _filled(W, 40, 2, D, dtype, 64, 22)
    at = torch.randint(0, 240, (W, 1, 4), generator=g)
    at[:, :, 0] = at[:, :, 0] % 200                      # a prefix's key, and one of the sequence's own
    at[:, :, 1] = 200 + at[:, :, 1] % 40
    keys = [torch.cat([pv[0][0], k]) for k, _ in ov]
    values = [torch.cat([pv[0][1], v]) for _, v in ov]
    q = torch.stack([torch.stack([keys[b][at[b, 0, h], h // 2] for h in range(4)]) for b in range(W)])[:, None]
    q = (q / q.norm(dim=-1, keepdim=True) * size * math.sqrt(D) / 8).to(dtype)
    # what the others' probabilities come to, from the values that the call is given
    x = torch.stack([torch.einsum("hd,thd->ht", q[b, 0].double(), keys[b].double().repeat_interleave(2, 1)) for b in range(W)]) / math.sqrt(D)
    best = x.gather(2, at.view(W, 4, 1))
    rest = (x.scatter(2, at.view(W, 4, 1), -math.inf) - best).exp().sum(2)
    sure = rest < 1e-8                                   # (a longer key of nearly the same direction may pass it)
    assert sure.float().mean() > 0.6
    out = axs_cache_shared_attention_unified(q.to(DEV), prefix, torch.tensor([200], device=DEV), cache,
                                             torch.full((W,), 40, device=DEV))[:, 0].cpu()
    want = torch.stack([torch.stack([values[b][at[b, 0, h], h // 2] for h in range(4)]) for b in range(W)])
    for h in range(4):
        assert ref.rel(out[:, h][sure[:, h]], want[:, h][sure[:, h]]) <= _bound(dtype), h


def test_a_gradient_or_tangent_of_no_operator_is_dropped():
    import torch.autograd.forward_ad as fwAD

    from axs.unified import axs_beam_select_unified, axs_cache_shared_attention_unified

    prefix, _ = _filled(1, 40, 2, 32, torch.float32, 64, 1)
    cache, _ = _filled(3, 40, 2, 32, torch.float32, 64, 2)
    n1, n3 = torch.tensor([40], device=DEV), torch.full((3,), 40, device=DEV)
    q = torch.randn(3, 1, 4, 32, generator=_gen(1)).to(DEV)
    z, s = torch.randn(2, 3, 10, generator=_gen(2)).to(DEV), torch.zeros(2, 3, device=DEV)
    attend = lambda x: axs_cache_shared_attention_unified(x, prefix, n1, cache, n3)   # noqa: E731
    recorded = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        attend(recorded)
    with torch.no_grad():
        assert torch.equal(attend(recorded), attend(q))
    assert torch.equal(attend(recorded.detach()), attend(q))
    with fwAD.dual_level():
        for call, x in ((attend, q), (lambda x: axs_beam_select_unified(x, s), z), (lambda x: axs_beam_select_unified(z, x), s)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call(fwAD.make_dual(x, torch.ones_like(x)))


# ---- copies ------------------------------------------------------------------------


@pytest.mark.parametrize("in_place", [True, False])
def test_copies_of_sequences_that_start_past_32_bits(in_place):
    """Five sequences of 1.1e9 bytes of key codes each: the third starts past 2^31 bytes, the fifth past 2^32."""
    from axs.unified import AXSKVCacheUnified, axs_cache_copy_unified

    blocks, D, B = 137_500, 256, 5
    assert 2 * blocks * 32 * D > 1 << 31 and 4 * blocks * 32 * D > 1 << 32
    g = torch.Generator(device=DEV).manual_seed(3)
    sizes = [((blocks, 32, D), torch.int8), ((blocks,), torch.float32), ((blocks, D, 32), torch.int8), ((blocks,), torch.float32),
             ((32, D), torch.bfloat16), ((32, D), torch.bfloat16)]
    big = AXSKVCacheUnified(*(torch.empty(B, 1, *s, dtype=t, device=DEV) for s, t in sizes))
    for x in big:
        for y in x:
            y.random_(-127, 128, generator=g)
    n = 32 * blocks - 3
    source = [4, 0, 3, 2, 1]
    target = big if in_place else AXSKVCacheUnified(*(torch.zeros_like(x) for x in big))
    old = [x.clone() for x in big]
    axs_cache_copy_unified(big, torch.tensor(source, device=DEV), torch.full((B,), n, device=DEV), None if in_place else target)
    for i, p in enumerate(source):
        for x, y in zip(target[:4], old):
            assert torch.equal(x[i], y[p])
        for x, y in zip(target[4:], old[4:]):
            assert torch.equal(x[i, :, :29], y[p, :, :29])
            assert torch.equal(x[i, :, 29:], y[i, :, 29:] if in_place else torch.zeros_like(y[i, :, 29:]))
