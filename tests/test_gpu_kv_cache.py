"""The 8-bit cache on the GPU: codes and scales bit for bit those of the block
formula, attention over it against the 64-bit form on the values it stands for.

Attention's error: the query and the probabilities go in as f16 (11 bits; two
terms for float32), both small beside the output's rounding: float32 outputs
within 5e-6 (exponents of about 20 in float32, 2^-24 * 20, twice), bfloat16 and
float16 within 2 u.
"""
from __future__ import annotations

import math

import pytest
import torch

import decoder_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _bound(dt):
    return 5e-6 if dt == torch.float32 else 2 * ref.U[dt]


def _tokens(B, n, H, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + B + n)
    return tuple((torch.randn(B, n, H, D, generator=g) * torch.rand(1, n, H, 1, generator=g).exp()).to(DEV, dtype)
                 for _ in range(2))


def _filled(B, n, H, D, dtype, capacity=None, seed=0):
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified

    cache = AXSKVCacheUnified.empty(B, H, D, capacity or n, dtype, DEV)
    k, v = _tokens(B, n, H, D, dtype, seed)
    if n:
        axs_cache_append_unified(cache, k, v, torch.zeros(B, dtype=torch.int64, device=DEV))
    return cache, k, v


def _codes(cache, b, n):
    """Codes (n, H, D) and scales (blocks, H) of keys and values of sequence b."""
    nb = -(-n // 32)
    k = cache.k_codes[b, :, :nb].permute(1, 2, 0, 3).flatten(0, 1)[:n]
    v = cache.v_codes[b, :, :nb].permute(1, 3, 0, 2).flatten(0, 1)[:n]
    return (k.cpu(), cache.k_scales[b, :, :nb].T.cpu()), (v.cpu(), cache.v_scales[b, :, :nb].T.cpu())


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,n,H,D", [(1, 1, 1, 16), (2, 31, 2, 64), (1, 32, 1, 128), (3, 33, 2, 80), (2, 200, 3, 256),
                                     (1, 64, 4, 96)])
def test_append_and_read(B, n, H, D, dtype):
    from axs.unified import axs_cache_read_unified

    cache, k, v = _filled(B, n, H, D, dtype)
    first = torch.arange(B, device=DEV) - 2
    rk, rv = axs_cache_read_unified(cache, first, n + 5)
    for b in range(B):
        for x, (codes, scales), got in ((k, _codes(cache, b, n)[0], rk), (v, _codes(cache, b, n)[1], rv)):
            want, s = ref.quantize_tokens(x[b])
            assert torch.equal(codes, want) and torch.equal(scales, s)
            window = torch.zeros(n + 5, H, D)
            at = int(first[b])
            lo, hi = max(at, 0), min(at + n + 5, n)
            window[lo - at:hi - at] = ref.cache_values(x[b])[lo:hi]
            assert torch.equal(got[b].cpu(), window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_any_split_into_calls_gives_the_same_cache(dtype):
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified

    n, H, D = 150, 2, 48
    whole, k, v = _filled(2, n, H, D, dtype, 160)
    for parts in ([1] * n, [40, 1, 1, 70, 38], [31, 1, 32, 33, 53], [5, 100, 45]):
        cache = AXSKVCacheUnified.empty(2, H, D, 160, dtype, DEV)
        at = 0
        for p in parts:
            axs_cache_append_unified(cache, k[:, at:at + p], v[:, at:at + p],
                                     torch.full((2,), at, device=DEV, dtype=torch.int32))
            at += p
        for x, y in zip(cache[:4], whole[:4]):
            assert torch.equal(x, y), parts
        assert torch.equal(cache.k_tail[:, :, :n % 32], whole.k_tail[:, :, :n % 32])
        assert torch.equal(cache.v_tail[:, :, :n % 32], whole.v_tail[:, :, :n % 32])


def test_ragged_starts_rewinding_and_the_end():
    from axs.unified import axs_cache_append_unified

    cache, k, v = _filled(4, 70, 1, 32, torch.float32, 96)
    before = [x.clone() for x in cache]
    more_k, more_v = _tokens(4, 40, 1, 32, torch.float32, 9)
    # back to a block's first token, on from the end, past the capacity, outside the cache
    starts = torch.tensor([32, 70, 96, -1], device=DEV)
    axs_cache_append_unified(cache, more_k, more_v, starts)
    a = torch.cat([k[0, :32], more_k[0]])
    assert torch.equal(_codes(cache, 0, 72)[0][0], ref.quantize_tokens(a)[0])
    b = torch.cat([k[1], more_k[1]])[:96]   # what does not fit is dropped
    assert torch.equal(_codes(cache, 1, 96)[0][0], ref.quantize_tokens(b)[0])
    for x, y in zip(cache, before):
        assert torch.equal(x[2:], y[2:])


def test_zeros_extremes_and_bad_values():
    from axs.unified import axs_cache_attention_unified, axs_cache_append_unified, AXSKVCacheUnified

    cache = AXSKVCacheUnified.empty(1, 1, 16, 128, torch.float32, DEV)
    k, v = _tokens(1, 128, 1, 16, torch.float32)
    k[0, :32], v[0, :32] = 0, 3e38
    k[0, 32:64] *= 1e-30
    v[0, 100, 0, 3] = math.nan      # the last block's values
    axs_cache_append_unified(cache, k, v, torch.zeros(1, dtype=torch.int64, device=DEV))
    for x, (codes, scales) in zip((k, v), _codes(cache, 0, 128)):
        want, s = ref.quantize_tokens(x[0])
        assert torch.equal(codes, want) and torch.equal(scales.isnan(), s.isnan())
        assert torch.equal(scales.nan_to_num(), s.nan_to_num())
    q = torch.randn(1, 1, 1, 16, device=DEV)
    assert axs_cache_attention_unified(q, cache, torch.tensor([96], device=DEV)).isfinite().all()
    assert axs_cache_attention_unified(q, cache, torch.tensor([97], device=DEV)).isnan().all()
    # of two queries only the second sees the bad block
    two = axs_cache_attention_unified(q.expand(1, 2, 1, 16), cache, torch.tensor([97], device=DEV))
    assert two[0, 0].isfinite().all() and two[0, 1].isnan().all()


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,Tq,Hq,H,D,lengths", [
    (1, 1, 1, 1, 16, [1]), (2, 1, 8, 2, 64, [31, 33]), (3, 1, 8, 1, 128, [0, 300, 64]), (2, 5, 4, 2, 80, [5, 129]),
    (1, 1, 32, 4, 96, [777]), (2, 3, 6, 2, 256, [2, 1000]), (1, 40, 3, 1, 192, [100]), (4, 2, 2, 1, 112, [1, 2, 3, 4]),
    (1, 1, 4, 1, 128, [9000]), (2, 5, 16, 4, 128, [700, 5]), (1, 3, 8, 2, 64, [5000]), (40, 1, 28, 7, 64, list(range(1, 241, 6))),
])
def test_attention(B, Tq, Hq, H, D, lengths, dtype):
    from axs.unified import axs_cache_attention_unified

    n = max(max(lengths), 1)
    cache, k, v = _filled(B, n, H, D, dtype, n + 40)
    q = torch.randn(B, Tq, Hq, D, generator=torch.Generator().manual_seed(7)).to(DEV, dtype)
    out = axs_cache_attention_unified(q, cache, torch.tensor(lengths, device=DEV))
    assert out.dtype == dtype and out.shape == q.shape
    for b, m in enumerate(lengths):
        # the blocks hold all n tokens; a query sees the first m
        kv, vv = ref.cache_values(k[b])[:m], ref.cache_values(v[b])[:m]
        want = ref.attention(q[b:b + 1], kv[None], vv[None], causal=True)
        assert ref.rel(out[b:b + 1], want) <= _bound(dtype), (b, m)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_scale_large_and_small_queries_and_layout(dtype):
    from axs.unified import axs_cache_attention_unified

    cache, k, v = _filled(1, 100, 2, 64, dtype)
    n = torch.tensor([100], device=DEV, dtype=torch.int32)
    base = torch.randn(1, 4, 1, 65, generator=torch.Generator().manual_seed(7))
    kv, vv = (ref.cache_values(x[0])[None] for x in (k, v))
    for size, scale in ((1e-3, None), (30.0, 0.02), (2000.0, 1e-4), (1.0, -0.3), (1.0, 0.0)):
        q = (base * size).to(DEV, dtype).transpose(1, 2)[..., 1:]   # (1, 1, 4, 64), unaligned
        out = axs_cache_attention_unified(q, cache, n, scale)
        assert ref.rel(out, ref.attention(q, kv, vv, scale=scale)) <= _bound(dtype) * 2, (size, scale)


def test_past_32_bits():
    """Codes that start past 2^31 bytes into the cache."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_attention_unified, axs_cache_read_unified

    H, D, n = 4, 256, 2_200_000     # 2.25e9 bytes of key codes
    cache = AXSKVCacheUnified.empty(1, H, D, n, torch.bfloat16, DEV)
    k, v = _tokens(1, 50, H, D, torch.bfloat16)
    at = cache.max_tokens - 64
    starts = torch.tensor([at], device=DEV)
    axs_cache_append_unified(cache, k, v, starts)
    rk, rv = axs_cache_read_unified(cache, starts, 50)
    assert torch.equal(rk[0].cpu(), ref.cache_values(k[0])) and torch.equal(rv[0].cpu(), ref.cache_values(v[0]))
    # a query along one key far out of the others' reach takes its value
    q = (k[:, 49:50].float() * 40).to(torch.bfloat16)
    out = axs_cache_attention_unified(q, cache, starts + 50)
    assert ref.rel(out, ref.cache_values(v[0])[49:50][None]) <= 2 * ref.U[torch.bfloat16]


def test_streams_and_graph():
    from axs.unified import axs_cache_append_unified, axs_cache_attention_unified

    cache, k, v = _filled(3, 500, 2, 64, torch.float32, 600)
    q = torch.randn(3, 1, 8, 64, device=DEV)
    n = torch.tensor([500, 100, 321], device=DEV)
    want = axs_cache_attention_unified(q, cache, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = axs_cache_attention_unified(q, cache, n)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    new = torch.randn(3, 1, 2, 64, device=DEV)
    with torch.cuda.graph(graph):
        axs_cache_append_unified(cache, new, new, n)
        out = axs_cache_attention_unified(q, cache, n + 1)
    for i in range(3):
        new.copy_(torch.randn(3, 1, 2, 64, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        axs_cache_append_unified(cache, new, new, n)
        assert torch.equal(got, axs_cache_attention_unified(q, cache, n + 1))


def test_refusals():
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_attention_unified, axs_cache_read_unified

    c, k, v = _filled(2, 40, 2, 32, torch.float32)
    n = torch.tensor([40, 40], device=DEV)
    q = torch.zeros(2, 1, 4, 32, device=DEV)
    bad_dim = AXSKVCacheUnified.empty(2, 2, 24, 40, torch.float32, DEV)
    for bad in (lambda: axs_cache_attention_unified(q[..., :16], c, n), lambda: axs_cache_attention_unified(q[:1], c, n),
                lambda: axs_cache_attention_unified(q[:, :, :3], c, n), lambda: axs_cache_attention_unified(q.half(), c, n),
                lambda: axs_cache_attention_unified(q, c, n[:1]), lambda: axs_cache_attention_unified(q, c, n.float()),
                lambda: axs_cache_attention_unified(q, c, n, math.inf), lambda: axs_cache_attention_unified(q, c, n.cpu()),
                lambda: axs_cache_attention_unified(q, c._replace(k_codes=c.k_codes[:, :, :1]), n),
                lambda: axs_cache_attention_unified(q, c._replace(v_scales=c.v_scales.double()), n),
                lambda: axs_cache_attention_unified(q, c._replace(v_codes=c.v_codes.transpose(3, 4)), n),
                lambda: axs_cache_append_unified(c, k[..., :16], v[..., :16], n), lambda: axs_cache_append_unified(c, k, v[:, :3], n),
                lambda: axs_cache_append_unified(c, k.half(), v.half(), n), lambda: axs_cache_append_unified(c, k, v, n[:1]),
                lambda: axs_cache_append_unified(bad_dim, k[..., :24], v[..., :24], n),
                lambda: axs_cache_read_unified(c, n, -1), lambda: axs_cache_read_unified(c, n[:1], 1)):
        with pytest.raises(RuntimeError):
            bad()


def test_a_cache_without_blocks():
    """Reading gives 0, appending drops everything, attention sees nothing."""
    from axs.unified import AXSKVCacheUnified, axs_cache_append_unified, axs_cache_attention_unified, axs_cache_read_unified

    cache = AXSKVCacheUnified.empty(2, 2, 32, 0, torch.float32, DEV)
    x = torch.ones(2, 3, 2, 32, device=DEV)
    n = torch.tensor([0, 5], device=DEV)
    axs_cache_append_unified(cache, x, x, n)
    for count in (1, 40):
        for y in axs_cache_read_unified(cache, n - 2, count):
            assert y.shape == (2, count, 2, 32) and not y.any()
    assert not axs_cache_attention_unified(x, cache, n).any()


def test_reading_outside_the_blocks():
    from axs.unified import axs_cache_read_unified

    cache, k, v = _filled(1, 64, 2, 32, torch.float32)
    for first, count in ((-100, 90), (64, 33), (1000, 5), (-3, 70)):
        for x, y in zip((k, v), axs_cache_read_unified(cache, torch.tensor([first], device=DEV), count)):
            want = torch.zeros(count, 2, 32)
            lo, hi = max(first, 0), min(first + count, 64)
            if lo < hi:
                want[lo - first:hi - first] = ref.cache_values(x[0])[lo:hi]
            assert torch.equal(y[0].cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e30, 1e-20, 1e-26, 1e-28, 1e-30])
def test_values_of_any_size(size, dtype):
    """Sums over large values stay finite and those over small ones keep their digits."""
    from axs.unified import axs_cache_attention_unified, axs_cache_append_unified, AXSKVCacheUnified

    for Tq, n in ((1, 300), (3, 9000)):
        cache = AXSKVCacheUnified.empty(1, 2, 64, n, dtype, DEV)
        k, v = _tokens(1, n, 2, 64, dtype)
        v = (v.float() * size).to(dtype)
        axs_cache_append_unified(cache, k, v, torch.zeros(1, dtype=torch.int64, device=DEV))
        q = torch.randn(1, Tq, 8, 64, generator=torch.Generator().manual_seed(7)).to(DEV, dtype)
        out = axs_cache_attention_unified(q, cache, torch.tensor([n], device=DEV))
        want = ref.attention(q, ref.cache_values(k[0])[None], ref.cache_values(v[0])[None], causal=True)
        assert ref.rel(out.double() / size, want / size) <= _bound(dtype), (n, Tq)
