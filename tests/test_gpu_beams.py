"""Beam search on the GPU: the selection against its 64-bit form, copies of cached
sequences bit for bit, attention over a shared prefix against the 64-bit form on the
values that the caches stand for, and the three together.

Attention's bound is the cache attention's: float32 outputs within 5e-6, bfloat16 and
float16 within 2 u.
"""
from __future__ import annotations

import math

import pytest
import torch

import beam_ref
import decoder_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- selection ---------------------------------------------------------------------


def _check_select(logits, scores, finished=None, end=None, count=None):
    from axs.unified import axs_beam_select_unified

    got = axs_beam_select_unified(logits, scores, finished, end, count)
    want = beam_ref.select(logits, scores, finished, end, count)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int64
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    s = got[0].double().cpu()
    assert torch.equal(s.isnan(), want[0].isnan()) and torch.equal(s == -math.inf, want[0] == -math.inf)
    some = want[0].isfinite()
    assert ((s - want[0]).abs()[some] <= beam_ref.select_bound(want[0], logits.shape[-1])[some]).all()


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("G,W,V,count", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 3), (1, 4, 256, 4), (3, 5, 1000, 10), (2, 48, 513, 96),
                                         (1, 64, 4097, 128), (5, 2, 50001, 4), (1, 1024, 33, 128), (2, 8, 32000, 16),
                                         (40, 3, 255, None), (1, 2, 131073, 2)])
def test_select(G, W, V, count, dtype):
    g = _gen(G + W + V)
    logits = (2.5 * torch.randn(G, W, V, generator=g)).to(DEV, dtype)
    scores = -5 * torch.rand(G, W, generator=g).to(DEV)
    _check_select(logits, scores, count=count)
    finished = (torch.rand(G, W, generator=g) < 0.3).to(DEV)
    _check_select(logits, scores, finished, V // 2, count)
    _check_select(logits, scores, torch.ones_like(finished), V - 1, count)
    # one prompt's first step: one beam counts
    scores[:, 1:] = -math.inf
    _check_select(logits, scores, count=count)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("G,W,V,count", [(1, 1, 2000, 128), (2, 8, 5000, 16), (1, 40, 3001, 100)])
def test_equal_candidates_stand_in_order(G, W, V, count, dtype):
    g = _gen(V)
    scores = torch.zeros(G, W, device=DEV)
    _check_select(torch.zeros(G, W, V, device=DEV, dtype=dtype), scores, count=count)
    # few different values, the same ones in every row: equal sums, beams that are copies of each other
    row = torch.randint(0, 3, (V,), generator=g).to(DEV, dtype)
    _check_select(row.expand(G, W, V), scores - 1.5, count=count)
    _check_select(row.expand(G, W, V).contiguous(), scores, torch.arange(W, device=DEV).expand(G, W) % 3 == 1, 7, count)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_masked_candidates(dtype):
    g = _gen(3)
    logits = torch.randn(4, 3, 700, generator=g).to(DEV, dtype)
    scores = -torch.rand(4, 3, generator=g).to(DEV)
    logits[0, :, 10:] = -math.inf                    # fewer candidates than asked for
    logits[1, 1] = -math.inf                         # a row that offers nothing
    logits[2] = torch.finfo(dtype).min               # masked by the type's lowest value: all alike
    logits[2, 0, 600] = 0
    logits[3, :, 1:] = torch.finfo(dtype).min
    _check_select(logits, scores, count=40)
    logits[:] = -math.inf
    _check_select(logits, scores, count=40)
    _check_select(logits, torch.full_like(scores, -math.inf), count=5)
    finished = torch.zeros(4, 3, dtype=torch.bool, device=DEV)
    finished[1, 2] = finished[3] = True
    _check_select(logits, scores, finished, 699, 4)


def test_bad_values_stay_in_their_sequence():
    logits = torch.randn(6, 4, 3000, generator=_gen(4)).to(DEV)
    scores = -torch.rand(6, 4, generator=_gen(5)).to(DEV)
    logits[0, 2, 2999] = math.nan
    logits[1, 0, 0] = math.inf
    scores[2, 3] = math.nan
    scores[3, 0] = math.inf
    # not read: beams that have ended or offer nothing
    logits[4, 1], scores[4, 1] = math.nan, -math.inf
    finished = torch.zeros(6, 4, dtype=torch.bool, device=DEV)
    finished[5, 2], logits[5, 2] = True, math.nan
    _check_select(logits, scores, finished, 17, 9)
    finished[2, 3] = True
    _check_select(logits, scores, finished, 17, 9)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_wide_scores(dtype):
    """Scores and logits far apart, and as near as their types allow."""
    g = _gen(6)
    logits = torch.randn(3, 5, 2222, generator=g).to(DEV, dtype)
    scores = torch.tensor([0.0, -1e30, -3e4, -1e-30, -0.0], device=DEV).expand(3, 5).contiguous()
    logits[1] *= 100
    logits[2] = logits[2] / 100 + 30
    scores[2] = -0.37 * torch.arange(5, device=DEV)
    _check_select(logits, scores, count=128)
    _check_select(logits, -100 - torch.rand(3, 5, generator=g).to(DEV), count=77)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_select_layouts(dtype):
    base = torch.randn(3, 2, 6, 1003, generator=_gen(7)).to(DEV, dtype)
    scores = -torch.rand(6, 3, generator=_gen(8)).to(DEV)
    for logits, s in ((base[:, 0].transpose(0, 1), scores),                 # (6, 3, 1003), rows at odd places
                      (base[:, 1, :, 3:998].transpose(0, 1), scores),
                      (base[0, 0].expand(2, 6, 1003), scores.view(2, 9)[:, :6]),
                      (base[:, 0].permute(2, 0, 1)[..., :4], -torch.rand(1003, 3, generator=_gen(9)).to(DEV))):
        _check_select(logits, s)


def test_select_refusals():
    from axs.unified import axs_beam_select_unified as select

    z, s = torch.zeros(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    f = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    for bad in (lambda: select(z[0], s), lambda: select(z, s[:1]), lambda: select(z, s.double()), lambda: select(z.double(), s),
                lambda: select(z, s.cpu()), lambda: select(z, s, f), lambda: select(z, s, f, 10), lambda: select(z, s, f, -1),
                lambda: select(z, s, f[:1], 1), lambda: select(z, s, f.int(), 1), lambda: select(z, s, f.cpu(), 1),
                lambda: select(z, s, count=0), lambda: select(z, s, count=129), lambda: select(z[:, :0], s[:, :0]),
                lambda: select(z[..., :0], s), lambda: select(z.clone().requires_grad_(), s),
                lambda: select(torch.zeros(1, 1025, 2, device=DEV), torch.zeros(1, 1025, device=DEV))):
        with pytest.raises(RuntimeError):
            bad()
    empty = select(z[:0], s[:0])
    assert [x.shape for x in empty] == [(0, 3)] * 3


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("G,W,V,count", [(1, 1000, 9000, 5), (2, 600, 9000, 128)])
def test_select_over_many_segments(G, W, V, count, dtype):
    """More segments than are looked at in one go, and as many equal ones."""
    logits = torch.randn(G, W, V, generator=_gen(V)).to(DEV, dtype)
    scores = -torch.rand(G, W, generator=_gen(W)).to(DEV)
    _check_select(logits, scores, count=count)
    # all alike: the first tokens of the first beam
    got = axs_select(torch.full_like(logits, 0.5), torch.zeros_like(scores), count)
    assert not got[1].any() and torch.equal(got[2].cpu(), torch.arange(count).expand(G, count))


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_select_among_many_equal_tokens(dtype):
    V = 300000
    logits = torch.zeros(2, 1, V, device=DEV, dtype=dtype)
    got = axs_select(logits, torch.zeros(2, 1, device=DEV), 128)
    assert not got[1].any() and torch.equal(got[2].cpu(), torch.arange(128).expand(2, 128))
    # the best of them at the end, and one of each few hundred
    logits[0, 0, -200:] = 1
    logits[1, 0, 5::601] = 1
    got = axs_select(logits, torch.zeros(2, 1, device=DEV), 128)
    assert torch.equal(got[2].cpu(), torch.stack([torch.arange(V - 200, V - 72), 5 + 601 * torch.arange(128)]))


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("W,ended,V,count", [(8, 4, 5000, 16), (80, 70, 900, 100), (40, 39, 40000, 128)])
def test_more_equal_tokens_than_are_listed_behind_ended_beams(W, ended, V, count, dtype):
    """The best segments are ended beams', which have no logits to wait for; of those behind them more tokens are
    alike than one list holds, so a second choice follows the first at once."""
    G = 24
    logits = torch.zeros(G, W, V, device=DEV, dtype=dtype)
    finished = torch.zeros(G, W, dtype=torch.bool, device=DEV)
    finished[:, :ended] = True
    scores = torch.where(finished, 0.0, -1.0)
    want = beam_ref.select(logits[:1], scores[:1], finished[:1], 9, count)
    for _ in range(5):
        got = _beam_select(logits, scores, finished, 9, count)
        assert torch.equal(got[1].cpu(), want[1].expand(G, -1)) and torch.equal(got[2].cpu(), want[2].expand(G, -1))
        assert ((got[0].cpu() - want[0]).abs() <= beam_ref.select_bound(want[0], V)).all()


def _beam_select(*args):
    from axs.unified import axs_beam_select_unified

    return axs_beam_select_unified(*args)


def axs_select(logits, scores, count):
    from axs.unified import axs_beam_select_unified

    return axs_beam_select_unified(logits, scores, count=count)


# ---- copies ------------------------------------------------------------------------


def _random_cache(B, H, D, tokens, dtype, seed):
    """Any bits will do: a copy does not look at them."""
    from axs.unified import AXSKVCacheUnified

    g, nb = _gen(seed), -(-tokens // 32)
    codes = [torch.randint(-127, 128, (B, H, nb, *x), generator=g, dtype=torch.int8) for x in ((32, D), (D, 32))]
    scales = [torch.rand(B, H, nb, generator=g) for _ in range(2)]
    tails = [torch.randn(B, H, 32, D, generator=g).to(dtype) for _ in range(2)]
    return AXSKVCacheUnified(*(x.to(DEV) for x in (codes[0], scales[0], codes[1], scales[1], *tails)))


def _check_copy(cache, sources, lengths, target=None):
    from axs.unified import axs_cache_copy_unified

    want = beam_ref.copy(cache, sources, lengths, target)
    before = [x.clone() for x in cache]
    axs_cache_copy_unified(cache, sources, lengths, target)
    for x, y in zip(cache if target is None else target, want):
        assert torch.equal(x.cpu(), y)
    if target is not None and target is not cache:
        assert all(torch.equal(x, y) for x, y in zip(cache, before))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,W,H,D,tokens", [(1, 1, 1, 16, 32), (1, 4, 2, 64, 70), (3, 5, 1, 80, 200), (2, 17, 3, 128, 96), (4, 2, 2, 256, 40),
                                            (1, 70, 1, 48, 130), (1, 300, 2, 16, 64), (1, 1100, 1, 16, 33)])
def test_copy_in_place(G, W, H, D, tokens, dtype):
    g = _gen(G + W)
    B = G * W
    for case in range(4):
        cache = _random_cache(B, H, D, tokens, dtype, case)
        if case == 0:      # a cycle through all
            src = torch.arange(1, W + 1).remainder(W).expand(G, W)
        elif case == 1:    # any beam's parent, some twice
            src = torch.randint(0, W, (G, W), generator=g)
        elif case == 2:    # some left alone
            src = torch.randint(-2, W + 3, (G, W), generator=g)
        else:              # everybody from the last
            src = torch.full((G, W), W - 1)
        lengths = torch.randint(-3, tokens + 40, (B,), generator=g)
        lengths[::3] = lengths[::3].clamp(0, tokens) // 32 * 32
        lengths[0] = (0, 1, tokens, 33)[case]
        _check_copy(cache, src.to(DEV), lengths.to(DEV))
        if G == 1:
            _check_copy(cache, src.flip(1)[0].to(DEV, torch.int32), lengths.to(DEV, torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("G,n,W,H,D,tokens,room", [(1, 1, 1, 1, 16, 32, 32), (2, 1, 8, 2, 80, 100, 200), (1, 3, 70, 1, 64, 200, 65),
                                                   (2, 5, 2, 3, 128, 33, 64), (1, 2, 700, 1, 16, 64, 40)])
def test_copy_to_another_cache(G, n, W, H, D, tokens, room, dtype):
    g = _gen(G + W + n)
    cache, target = _random_cache(G * n, H, D, tokens, dtype, 1), _random_cache(G * W, H, D, room, dtype, 2)
    lengths = torch.randint(0, tokens + 1, (G * n,), generator=g)
    lengths[0] = tokens
    _check_copy(cache, torch.randint(-1, n + 1, (G, W), generator=g).to(DEV), lengths.to(DEV), target)
    _check_copy(cache, torch.randint(-1, G * n, (G * W,), generator=g).to(DEV), lengths.to(DEV), target)
    # a cache given as its own target is itself
    _check_copy(target, torch.arange(W - 1, -1, -1).expand(G, W).to(DEV), torch.full((G * W,), room, device=DEV), target)


def test_copies_of_nothing():
    from axs.unified import AXSKVCacheUnified, axs_cache_copy_unified

    cache = _random_cache(2, 1, 16, 64, torch.float32, 0)
    n = torch.tensor([64, 64], device=DEV)
    before = [x.clone() for x in cache]
    none = AXSKVCacheUnified.empty(2, 1, 16, 0, device=DEV)
    axs_cache_copy_unified(none, n * 0, n, cache)
    axs_cache_copy_unified(cache, n * 0, n, none)
    axs_cache_copy_unified(cache, torch.zeros(0, dtype=torch.int64, device=DEV), n, AXSKVCacheUnified.empty(0, 1, 16, 64, device=DEV))
    axs_cache_copy_unified(cache, torch.tensor([1, 0], device=DEV), n * 0)
    axs_cache_copy_unified(cache, torch.tensor([[0], [0]], device=DEV), n)
    assert all(torch.equal(x, y) for x, y in zip(cache, before))


def test_copied_sequences_go_on():
    """A copy's tail carries its partial block: appending and attending go on as in the original."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_attention_unified, axs_cache_copy_unified

    g = _gen(11)
    x = torch.randn(2, 45, 2, 64, generator=g).to(DEV)
    cache = AXSKVCacheUnified.empty(2, 2, 64, 96, torch.float32, DEV)
    n = torch.tensor([45, 45], device=DEV)
    axs_cache_append_unified(cache, x, x, n * 0)
    beams = AXSKVCacheUnified.empty(6, 2, 64, 128, torch.float32, DEV)
    axs_cache_copy_unified(cache, torch.zeros(2, 3, dtype=torch.int64, device=DEV), n, beams)
    new = torch.randn(6, 1, 2, 64, generator=g).to(DEV)
    axs_cache_append_unified(beams, new, new, n.repeat_interleave(3))
    q = torch.randn(6, 1, 4, 64, generator=g).to(DEV)
    out = axs_cache_attention_unified(q, beams, n.repeat_interleave(3) + 1)
    for b in range(6):
        kv = ref.cache_values(torch.cat([x[b // 3], new[b]]))[None]
        assert ref.rel(out[b:b + 1], ref.attention(q[b:b + 1], kv, kv)) <= 5e-6


def test_copy_past_32_bits():
    """Codes past 2^31 bytes, and sequences whose codes start there."""
    cache = _random_cache(2, 1, 256, 64, torch.bfloat16, 0)
    n = 4_400_000                     # 1.1e9 bytes of key codes a sequence
    from axs.unified import AXSKVCacheUnified, axs_cache_copy_unified

    big = AXSKVCacheUnified(*(torch.empty(2 if i < 4 else 2, 1, *x, dtype=t, device=DEV) for i, (x, t) in enumerate(
        [((n // 32, 32, 256), torch.int8), ((n // 32,), torch.float32), ((n // 32, 256, 32), torch.int8), ((n // 32,), torch.float32),
         ((32, 256), torch.bfloat16), ((32, 256), torch.bfloat16)])))
    last = n // 32 - 2
    for x, y in zip(big[:4], cache[:4]):
        x[:, :, last:] = y
    for x, y in zip(big[4:], cache[4:]):
        x.copy_(y)
    axs_cache_copy_unified(big, torch.tensor([1, 0], device=DEV), torch.full((2,), n - 1, device=DEV))
    for x, y in zip(big[:4], cache[:4]):
        assert torch.equal(x[:, :, last:], y.flip(0))
    assert torch.equal(big.k_tail[:, :, :31], cache.k_tail.flip(0)[:, :, :31])
    assert torch.equal(big.k_tail[:, :, 31:], cache.k_tail[:, :, 31:])


def test_copy_refusals():
    from axs.unified import axs_cache_copy_unified as copy

    c = _random_cache(4, 2, 32, 64, torch.float32, 0)
    s, n = torch.zeros(4, dtype=torch.int64, device=DEV), torch.full((4,), 64, device=DEV)
    part = type(c)(*(x[1:3] for x in c))
    wide = type(c)(*(torch.zeros(4097, *x.shape[1:], dtype=x.dtype, device=DEV) for x in c))
    for bad in (lambda: copy(c, s[:3], n), lambda: copy(c, s.view(1, 2, 2), n), lambda: copy(c, s, n[:2]),
                lambda: copy(c, s.float(), n), lambda: copy(c, s.cpu(), n), lambda: copy(c, s[:3].view(3, 1), n),
                lambda: copy(c, s, n, _random_cache(4, 1, 32, 64, torch.float32, 0)),
                lambda: copy(c, s, n, _random_cache(4, 2, 48, 64, torch.float32, 0)),
                lambda: copy(c, s, n, _random_cache(4, 2, 32, 64, torch.float16, 0)),
                lambda: copy(c, s[:2], n, part),                                      # memory of the cache's own
                lambda: copy(part, s, n[:2], c),
                lambda: copy(c, s, n, c._replace(k_tail=c.v_tail, v_tail=c.k_tail)),
                lambda: copy(c, s, n, c._replace(k_scales=c.k_scales.clone())),
                lambda: copy(wide, torch.zeros(4097, dtype=torch.int64, device=DEV),
                             torch.zeros(4097, dtype=torch.int64, device=DEV))):
        with pytest.raises(RuntimeError):
            bad()


# ---- attention over a shared prefix ------------------------------------------------------


def _tokens(B, n, H, D, dtype, seed):
    g = _gen(seed)
    return tuple((torch.randn(B, n, H, D, generator=g) * torch.rand(1, n, H, 1, generator=g).exp()).to(DEV, dtype)
                 for _ in range(2))


def _filled(B, n, H, D, dtype, capacity, seed):
    """A cache of n tokens a sequence, and what it stands for."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified

    cache = AXSKVCacheUnified.empty(B, H, D, capacity, dtype, DEV)
    k, v = _tokens(B, n, H, D, dtype, seed)
    axs_cache_append_unified(cache, k, v, torch.zeros(B, dtype=torch.int64, device=DEV))
    return cache, [(ref.cache_values(k[b]), ref.cache_values(v[b])) for b in range(B)]


def _bound(dt):
    return 5e-6 if dt == torch.float32 else 2 * ref.U[dt]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("P,W,Tq,Hq,H,D,np,n", [
    (1, 1, 1, 1, 1, 16, [1], [1]), (1, 4, 1, 8, 2, 64, [300], [3, 1, 33, 20]), (2, 3, 1, 4, 4, 128, [31, 64], [5] * 6),
    (2, 2, 2, 6, 2, 80, [100, 0], [2, 40, 2, 64]), (1, 20, 1, 16, 2, 128, [1000], list(range(1, 21))),
    (3, 8, 1, 8, 1, 96, [700, 33, 2000], [32] * 24), (1, 6, 5, 4, 2, 64, [129], [0, 1, 4, 5, 6, 70]),
    (1, 2, 7, 2, 1, 48, [3], [2, 5]), (2, 40, 1, 4, 1, 256, [200, 900], [9] * 80), (1, 33, 3, 2, 1, 192, [500], [40] * 33),
    (1, 64, 1, 32, 4, 128, [4000], [50] * 64), (1, 3, 1, 4, 2, 128, [9000], [300, 700, 1]), (12, 2, 1, 28, 7, 64, [257] * 12, [8] * 24),
    (70, 2, 1, 4, 2, 64, [40, 0, 33, 300, 1, 96, 64] * 10, [8, 1] * 70), (65, 20, 1, 2, 1, 112, [77] * 65, [3] * 1300),
    (5, 9, 2, 8, 2, 144, [0, 700, 31, 33, 64], [2] * 45),
])
def test_shared_attention(P, W, Tq, Hq, H, D, np, n, dtype):
    from axs.unified import axs_cache_shared_attention_unified

    prefix, pv = _filled(P, max(max(np), 1), H, D, dtype, max(np) + 40, 1)
    cache, ov = _filled(P * W, max(max(n), 1), H, D, dtype, max(n) + 3, 2)
    q = torch.randn(P * W, Tq, Hq, D, generator=_gen(7)).to(DEV, dtype)
    out = axs_cache_shared_attention_unified(q, prefix, torch.tensor(np, device=DEV), cache, torch.tensor(n, device=DEV))
    assert out.dtype == dtype and out.shape == q.shape
    want = beam_ref.shared_attention(q, pv, np, ov, n)
    for b in range(P * W):
        assert ref.rel(out[b], want[b]) <= _bound(dtype), b


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_shared_scale_size_and_layout(dtype):
    from axs.unified import axs_cache_shared_attention_unified

    prefix, pv = _filled(1, 200, 2, 64, dtype, 256, 3)
    cache, ov = _filled(9, 20, 2, 64, dtype, 32, 4)
    np, n = torch.tensor([200], device=DEV, dtype=torch.int32), torch.full((9,), 20, device=DEV, dtype=torch.int32)
    base = torch.randn(9, 8, 1, 65, generator=_gen(7))
    for size, scale in ((1e-3, None), (30.0, 0.02), (2000.0, 1e-4), (1.0, -0.3), (1.0, 0.0)):
        q = (base * size).to(DEV, dtype).transpose(1, 2)[..., 1:]   # unaligned
        out = axs_cache_shared_attention_unified(q, prefix, np, cache, n, scale)
        assert ref.rel(out, beam_ref.shared_attention(q, pv, [200], ov, [20] * 9, scale)) <= _bound(dtype) * 2, (size, scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,own", [(1e30, 1e30), (1e-20, 1e-20), (1e-28, 1e-28), (1e-30, 1.0), (1.0, 1e-30), (1e30, 1.0)])
@pytest.mark.parametrize("W", [2, 40])
def test_shared_values_of_any_size(size, own, W, dtype):
    """Large values stay finite and small ones keep their digits, whatever the other part's are."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_shared_attention_unified

    caches, values = [], []
    for B, n, s, seed in ((1, 1500, size, 5), (W, 40, own, 6)):
        cache = AXSKVCacheUnified.empty(B, 1, 64, n, dtype, DEV)
        k, v = _tokens(B, n, 1, 64, dtype, seed)
        v = (v.float() * s).to(dtype)
        axs_cache_append_unified(cache, k, v, torch.zeros(B, dtype=torch.int64, device=DEV))
        caches.append(cache)
        values.append([(ref.cache_values(k[b]), ref.cache_values(v[b])) for b in range(B)])
    q = torch.randn(W, 1, 4, 64, generator=_gen(8)).to(DEV, dtype)
    out = axs_cache_shared_attention_unified(q, caches[0], torch.tensor([1500], device=DEV), caches[1],
                                             torch.full((W,), 40, device=DEV))
    want = beam_ref.shared_attention(q, values[0], [1500], values[1], [40] * W)
    top = max(size, own)
    assert ref.rel(out.double() / top, want / top) <= _bound(dtype)


@pytest.mark.parametrize("D,blocks", [(128, 33000), (256, 16500)])
@pytest.mark.parametrize("W", [1, 24])
def test_shared_past_32_bits(W, D, blocks):
    """Prefixes and own tokens that lie more than 2^32 bytes into their caches."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_shared_attention_unified

    dt = torch.bfloat16
    prefix = AXSKVCacheUnified.empty(3, 12, D, 32 * blocks, dt, DEV)
    cache = AXSKVCacheUnified.empty(3 * W, 12, D, 32 * blocks // W, dt, DEV)
    assert prefix.k_codes[2].storage_offset() > 1 << 32 or prefix.k_codes.numel() > 1 << 32
    values = []
    for c, tokens, seed in ((prefix, 300, 3), (cache, 40, 4)):
        k, v = _tokens(c.k_codes.shape[0], tokens, 12, D, dt, seed)
        axs_cache_append_unified(c, k, v, torch.zeros(k.shape[0], dtype=torch.int64, device=DEV))
        values.append([(ref.cache_values(k[b]), ref.cache_values(v[b])) for b in range(k.shape[0])])
    np, n = torch.tensor([300, 7, 290], device=DEV), torch.full((3 * W,), 40, device=DEV)
    q = torch.randn(3 * W, 1, 12, D, generator=_gen(7)).to(DEV, dt)
    out = axs_cache_shared_attention_unified(q, prefix, np, cache, n)
    want = beam_ref.shared_attention(q, values[0], np.tolist(), values[1], n.tolist())
    assert ref.rel(out[-W:], want[-W:]) <= _bound(dt) and ref.rel(out[:W], want[:W]) <= _bound(dt)


@pytest.mark.parametrize("W", [2, 40])
def test_a_bad_block_counts_where_it_is_seen(W):
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_shared_attention_unified

    prefix, cache = (AXSKVCacheUnified.empty(B, 1, 32, 160, torch.float32, DEV) for B in (1, W))
    k, v = _tokens(1, 160, 1, 32, torch.float32, 9)
    v[0, 130, 0, 3] = math.nan
    axs_cache_append_unified(prefix, k, v, torch.zeros(1, dtype=torch.int64, device=DEV))
    ok, ov = _tokens(W, 70, 1, 32, torch.float32, 10)
    ok[1, 64:] = math.inf
    axs_cache_append_unified(cache, ok, ov, torch.zeros(W, dtype=torch.int64, device=DEV))
    q = torch.randn(W, 2, 2, 32, generator=_gen(8)).to(DEV)

    def call(np, n):
        return axs_cache_shared_attention_unified(q, prefix, torch.tensor([np], device=DEV), cache, torch.tensor(n, device=DEV))

    assert call(128, [64] * W).isfinite().all()
    assert call(129, [64] * W).isnan().all()
    out = call(128, [70] * W)           # the second sequence's last block
    assert out[1].isnan().all() and out[torch.arange(W) != 1].isfinite().all()
    out = call(128, [65] * W)           # seen by the last query alone
    assert out[1, 1].isnan().all() and out[1, 0].isfinite().all()
    out = call(129, [1] + [0] * (W - 1))   # a query that lies in the prefix, before the bad block
    assert out[0].isnan()[1].all() and out[1:, 0].isfinite().all() and out[1:, 1].isnan().all()


def test_shared_without_tokens():
    from axs.unified import AXSKVCacheUnified, axs_cache_attention_unified, axs_cache_shared_attention_unified

    q = torch.randn(6, 2, 4, 32, generator=_gen(1)).to(DEV)
    full, _ = _filled(2, 40, 2, 32, torch.float32, 64, 1)
    own, _ = _filled(6, 40, 2, 32, torch.float32, 64, 2)
    empty2, empty6 = (AXSKVCacheUnified.empty(B, 2, 32, 0, torch.float32, DEV) for B in (2, 6))
    zero2, zero6 = (torch.zeros(B, dtype=torch.int64, device=DEV) for B in (2, 6))
    n2, n6 = zero2 + 40, zero6 + 33
    call = axs_cache_shared_attention_unified
    assert not call(q, empty2, n2, empty6, n6).any()
    assert not call(q, full, zero2, own, zero6).any() and not call(q, full, zero2 - 5, own, zero6 - 1).any()
    alone = axs_cache_attention_unified(q, own, n6)
    assert torch.equal(call(q, empty2, n2, own, n6), alone)
    assert ref.rel(call(q, full, zero2, own, n6), alone) <= 5e-6
    # only the prefix: its last tokens are the queries, of three sequences each
    want = torch.cat([axs_cache_attention_unified(q[i::3], full, n2) for i in range(3)])
    got = call(q, full, n2, empty6, n6)
    assert ref.rel(torch.cat([got[i::3] for i in range(3)]), want) <= 5e-6
    assert call(q[:0], type(full)(*(x[:0] for x in full)), n2[:0], type(own)(*(x[:0] for x in own)), n6[:0]).shape == (0, 2, 4, 32)
    assert call(q[:, :0], full, n2, own, n6).shape == (6, 0, 4, 32)


def test_shared_refusals():
    from axs.unified import axs_cache_shared_attention_unified as call

    p, _ = _filled(2, 40, 2, 32, torch.float32, 64, 1)
    c, _ = _filled(6, 40, 2, 32, torch.float32, 64, 2)
    q = torch.zeros(6, 1, 4, 32, device=DEV)
    n2, n6 = torch.full((2,), 40, device=DEV), torch.full((6,), 40, device=DEV)
    half = type(p)(*(x.half() if i > 3 else x for i, x in enumerate(p)))
    five = type(c)(*(x[:5] for x in c))
    for bad in (lambda: call(q[:5], p, n2, five, n6[:5]), lambda: call(q, p, n2[:1], c, n6), lambda: call(q, p, n2, c, n6[:5]),
                lambda: call(q.half(), p, n2, c, n6), lambda: call(q, half, n2, c, n6), lambda: call(q[:, :, :3], p, n2, c, n6),
                lambda: call(q[..., :16], p, n2, c, n6), lambda: call(q, p, n2.float(), c, n6), lambda: call(q, p, n2.cpu(), c, n6),
                lambda: call(q, p, n2, c, n6, math.inf), lambda: call(q[0], p, n2, c, n6),
                lambda: call(q, type(p)(*(x[:, :1].contiguous() for x in p)), n2, c, n6)):
        with pytest.raises(RuntimeError):
            bad()


# ---- together ------------------------------------------------------------------------


def _step(state):
    """One step of a search: attention, new tokens' logits (from the attention's outputs), selection, caches after
    their parents."""
    from axs.unified import (axs_beam_select_unified, axs_cache_append_unified, axs_cache_copy_unified,
                             axs_cache_shared_attention_unified)

    G, W = state["scores"].shape
    new = state["embed"][state["tokens"].view(-1)].view(G * W, 1, 2, 64)
    axs_cache_append_unified(state["cache"], new, new, state["lengths"])
    state["lengths"] += 1
    q = new.repeat_interleave(2, 2)
    y = axs_cache_shared_attention_unified(q, state["prefix"], state["prefix_lengths"], state["cache"], state["lengths"])
    logits = (y.flatten(1) @ state["head"]).view(G, W, -1)
    scores, parents, tokens = axs_beam_select_unified(logits, state["scores"], state["finished"], 5)
    axs_cache_copy_unified(state["cache"], parents, state["lengths"])
    state["finished"].copy_(state["finished"].gather(1, parents) | (tokens == 5))
    state["scores"].copy_(scores)
    state["tokens"].copy_(tokens)
    return logits, parents


def _state(G, W, V):
    g = _gen(21)
    prefix, _ = _filled(G, 77, 2, 64, torch.float32, 96, 12)
    cache, _ = _filled(G * W, 1, 2, 64, torch.float32, 64, 13)
    return dict(prefix=prefix, cache=cache, prefix_lengths=torch.tensor([77, 50, 33][:G], device=DEV),
                lengths=torch.zeros(G * W, dtype=torch.int64, device=DEV),
                embed=torch.randn(V, 128, generator=g).to(DEV), head=(torch.randn(256, V, generator=g) / 4).to(DEV),
                scores=torch.tensor([0.0] + [-math.inf] * (W - 1), device=DEV).expand(G, W).contiguous(),
                finished=torch.zeros(G, W, dtype=torch.bool, device=DEV),
                tokens=torch.zeros(G, W, dtype=torch.int64, device=DEV))


def test_search_step_by_step():
    """Each step's choice is the 64-bit one's, and each beam's cache that of its own history."""
    from axs.unified import axs_cache_read_unified

    G, W, V = 3, 5, 90
    s = _state(G, W, V)
    history = torch.zeros(G, W, 0, dtype=torch.int64)
    for _ in range(40):
        before = s["scores"].clone(), s["finished"].clone()
        history = torch.cat([history, s["tokens"].cpu()[..., None]], 2)
        logits, parents = _step(s)
        want = beam_ref.select(logits, *before, 5)
        assert torch.equal(parents.cpu(), want[1]) and torch.equal(s["tokens"].cpu(), want[2])
        history = history.gather(1, parents.cpu()[..., None].expand_as(history))
    n = history.shape[2]
    k, v = axs_cache_read_unified(s["cache"], torch.zeros_like(s["lengths"]), n)
    for g in range(G):
        for w in range(W):
            if s["scores"][g, w] == -math.inf:
                continue
            want = ref.cache_values(s["embed"][history[g, w].to(DEV)].view(n, 2, 64))
            assert torch.equal(k[g * W + w].cpu(), want) and torch.equal(v[g * W + w].cpu(), want)


def test_streams_and_graph():
    """A search recorded once and replayed is the eager one; so is one on another stream."""
    want = _state(2, 4, 90)
    for _ in range(6):
        _step(want)
    side = _state(2, 4, 90)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(6):
            _step(side)
    stream.synchronize()
    s = _state(2, 4, 90)
    kept = {k: v.clone() for k, v in s.items() if isinstance(v, torch.Tensor)}
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        _step(s)
    warm.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(s)
    for k, v in kept.items():
        s[k].copy_(v)
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        torch.randn(1000, device=DEV).sum()
    for other in (side, s):
        for k in ("scores", "tokens", "finished", "lengths"):
            assert torch.equal(want[k], other[k]), k
        assert all(torch.equal(x[:, :, :1], y[:, :, :1]) for x, y in zip(want["cache"][:4], other["cache"][:4]))


def test_results_repeat():
    """The same calls give the same bits."""
    from axs.unified import axs_beam_select_unified, axs_cache_shared_attention_unified

    logits = torch.randn(4, 8, 20000, generator=_gen(1)).to(DEV, torch.bfloat16)
    scores = -torch.rand(4, 8, generator=_gen(2)).to(DEV)
    prefix, _ = _filled(2, 3000, 2, 64, torch.bfloat16, 3000, 1)
    cache, _ = _filled(40, 50, 2, 64, torch.bfloat16, 64, 2)
    q = torch.randn(40, 1, 16, 64, generator=_gen(3)).to(DEV, torch.bfloat16)
    np, n = torch.tensor([3000, 1234], device=DEV), torch.full((40,), 50, device=DEV)
    first = axs_beam_select_unified(logits, scores, count=64), axs_cache_shared_attention_unified(q, prefix, np, cache, n)
    for _ in range(3):
        again = axs_beam_select_unified(logits, scores, count=64), axs_cache_shared_attention_unified(q, prefix, np, cache, n)
        assert all(torch.equal(x, y) for x, y in zip(first[0], again[0])) and torch.equal(first[1], again[1])


def test_two_graphs_and_two_streams():
    """Two searches recorded apart and replayed by turns, then run at once on two streams: neither has the other's
    workspaces."""
    def run(a, n):
        for _ in range(n):
            _step(a)

    def state(seed):
        s = _state(2, 4, 90)
        s["embed"] = torch.randn(90, 128, generator=_gen(seed)).to(DEV)
        return s

    want = [state(40), state(41)]
    for w in want:
        run(w, 5)
    torch.cuda.synchronize()
    recorded, graphs = [state(40), state(41)], []
    for r in recorded:
        kept = {k: v.clone() for k, v in r.items() if isinstance(v, torch.Tensor)}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(r)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _step(r)
        graphs.append(graph)
        for k, v in kept.items():
            r[k].copy_(v)
    for _ in range(5):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
    at_once, streams = [state(40), state(41)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for a, stream in zip(at_once, streams):
            with torch.cuda.stream(stream):
                _step(a)
    torch.cuda.synchronize()
    for w, r, a in zip(want, recorded, at_once):
        for k in ("scores", "tokens", "finished", "lengths"):
            assert torch.equal(w[k], r[k]) and torch.equal(w[k], a[k]), k


# ---- in the framework's own paths ------------------------------------------------------


def _module(seed=0):
    import axs.unified as axu

    torch.manual_seed(seed)
    m = axu.AXSCausalSelfAttentionUnified(128, 4, 2).to(DEV).eval()
    return m, axu.rotary_table(32, 256, device=DEV)


@pytest.mark.parametrize("P,W,T", [(1, 4, 1), (3, 2, 1), (2, 3, 5)])
def test_decode_over_a_prefix(P, W, T):
    """A module's beams over a shared prompt: its parts, and as though each beam had its prompt's copy."""
    import axs.unified as axu

    m, table = _module()
    np = torch.tensor([64, 32, 0][:P], device=DEV)   # whole blocks: both caches hold the same codes and raw rows
    with torch.no_grad():
        prompts = torch.randn(P, 64, 128, generator=_gen(1)).to(DEV)
        prefix = m.new_cache(P, 64, device=DEV)
        m.decode(prompts, table, prefix, torch.zeros_like(np))
        cache, parts, whole = m.new_cache(P * W, 40, device=DEV), m.new_cache(P * W, 40, device=DEV), m.new_cache(P * W, 120, device=DEV)
        for b in range(P):
            own = m.new_cache(1, 64, device=DEV)
            if np[b]:
                m.decode(prompts[b:b + 1, :int(np[b])], table, own, torch.zeros(1, dtype=torch.int64, device=DEV))
            axu.axs_cache_copy_unified(own, torch.zeros(W, dtype=torch.int64, device=DEV), np[b:b + 1],
                                       axu.AXSKVCacheUnified(*(x[b * W:(b + 1) * W] for x in whole)))
        n = torch.zeros(P * W, dtype=torch.int64, device=DEV)
        long = np.repeat_interleave(W)
        for i in range(3):
            x = torch.randn(P * W, T, 128, generator=_gen(10 + i)).to(DEV)
            out = m.decode(x, table, cache, n, prefix, np)
            q, k, v = m._heads(x)
            q, k = axu.axs_rotary_unified(q, k, table, (long + n)[:, None] + torch.arange(T, device=DEV))
            axu.axs_cache_append_unified(parts, k, v, n)
            y = axu.axs_cache_shared_attention_unified(q, prefix, np, parts, n + T)
            assert torch.equal(out, m.out_proj(y.flatten(2)))
            axu.axs_cache_append_unified(whole, k, v, long + n)
            want = axu.axs_cache_attention_unified(q, whole, long + n + T)
            assert ref.rel(y, want) <= 2 * _bound(torch.float32)
            n += T
        with pytest.raises(ValueError):
            m.decode(x, table, cache, n, prefix)
        with pytest.raises(ValueError):
            m.decode(x, table, cache, n, None, np)
        with pytest.raises(ValueError):
            m.decode(x[1:], table, cache, n[1:], prefix, torch.zeros(4, dtype=torch.int64, device=DEV))
        with pytest.raises(ValueError):
            m.decode(x, table, cache, n, type(prefix)(*(t[:0] for t in prefix)), np)


class _Reader:
    """Logits that depend on each token of the history, read back from two caches: ids that the 8-bit codes hold
    exactly (at most 100 of them, half a step off by less than half)."""

    def __init__(self, G, W, V, starts, seed):
        from axs.unified import AXSKVCacheUnified, axs_cache_append_unified

        self.table = (2 * torch.randn(1009, V, generator=_gen(seed))).to(DEV)
        self.caches = [AXSKVCacheUnified.empty(G * W, h, 16, 80, torch.float32, DEV) for h in (1, 3)]
        self.prompt = torch.randint(0, V, (G, starts), generator=_gen(seed + 1))
        rows = self.prompt.repeat_interleave(W, 0).to(DEV).float()[..., None, None]
        for c in self.caches:
            x = rows.expand(-1, -1, c.k_codes.shape[1], 16).contiguous()
            axs_cache_append_unified(c, x, x, torch.zeros(G * W, dtype=torch.int64, device=DEV))

    def logits(self, history):
        h = torch.zeros(history.shape[0], dtype=torch.int64, device=history.device)
        for t in range(history.shape[1]):
            h = (31 * h + history[:, t] + 1) % 1009
        return self.table[h.to(DEV)]

    def __call__(self, tokens, starts):
        from axs.unified import axs_cache_append_unified, axs_cache_read_unified

        assert len(set(starts.tolist())) == 1
        n = int(starts[0]) + 1
        for c in self.caches:
            x = tokens.float()[..., None, None].expand(-1, -1, c.k_codes.shape[1], 16).contiguous()
            axs_cache_append_unified(c, x, -x, starts)
        ids = [axs_cache_read_unified(c, torch.zeros_like(starts), n) for c in self.caches]
        ids = [(k[..., 0, 3].round().long(), -v[..., -1, 7].round().long()) for k, v in ids]
        for k, v in ids[1:]:
            assert torch.equal(k, ids[0][0])
        return self.logits(ids[0][0])[:, None]


@pytest.mark.parametrize("G,W,V,steps,end,starts", [(1, 4, 60, 50, None, 0), (3, 5, 90, 40, 7, 0), (2, 3, 50, 45, 1, 29), (2, 1, 30, 9, 2, 3),
                                                    (1, 6, 3, 4, 0, 1), (1, 2, 10, 1, 4, 0)])
def test_beam_search(G, W, V, steps, end, starts):
    """The loop keeps histories, caches and ends together: the search over plain histories in 64 bits."""
    from axs.unified import axs_beam_search_unified

    m = _Reader(G, W, V, starts, 30 + V)
    start = torch.full((G * W,), starts, device=DEV)
    got = axs_beam_search_unified(m, m.logits(m.prompt), m.caches, W, steps, end, start if starts else None)
    assert int(start[0]) == starts
    scores = torch.tensor([0.0] + [-math.inf] * (W - 1)).expand(G, W)
    history, finished = m.prompt[:, None].expand(G, W, starts), torch.zeros(G, W, dtype=torch.bool)
    for _ in range(steps):
        z = m.logits(history.reshape(G * W, -1)).view(G, W, V)
        scores, parents, tokens = beam_ref.select(z, scores, finished, 0 if end is None else end)
        scores = scores.float()
        history = torch.cat([history.gather(1, parents[..., None].expand_as(history)), tokens[..., None]], 2)
        finished = finished.gather(1, parents) | (tokens == (-1 if end is None else end))
    assert torch.equal(got[1].cpu(), history[..., starts:])
    # a rounding and a sum's error a step
    some = scores.isfinite()
    assert torch.equal(got[0].cpu() == -math.inf, ~some)
    bound = steps * beam_ref.select_bound(scores.double(), V)
    assert ((got[0].cpu() - scores).abs()[some] <= bound[some]).all()


def test_beam_search_refusals():
    from axs.unified import axs_beam_search_unified as search

    z = torch.zeros(2, 9, device=DEV)
    for beams, steps in ((0, 3), (2, 0)):
        with pytest.raises(ValueError):
            search(None, z, [], beams, steps)
    for bad in (lambda: search(None, z[0], [], 2, 1), lambda: search(None, z, [], 129, 1), lambda: search(lambda t, s: z, z, [], 2, 3)):
        with pytest.raises((RuntimeError, IndexError)):
            bad()


def test_example_generates_with_beams():
    import importlib.util
    import os
    import sys

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "axs-6_amd", "examples", "distill_decoder.py")
    spec = importlib.util.spec_from_file_location("distill_decoder_beams", path)
    ex = sys.modules[spec.name] = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    torch.manual_seed(3)
    m = ex.Decoder(ex.Config(vocab=64, context=64, width=128), True).to(DEV)
    prompt = torch.randint(0, 64, (3, 21), generator=_gen(4)).to(DEV)
    scores, tokens = m.generate_beams(prompt, 40, 4)
    assert scores.shape == (3, 4) and tokens.shape == (3, 4, 61) and scores.isfinite().all()
    assert (scores[:, 1:] <= scores[:, :-1]).all() and torch.equal(tokens[..., :21], prompt[:, None].expand(3, 4, 21))
    assert len({tuple(x) for x in tokens.view(12, -1).tolist()}) == 12
