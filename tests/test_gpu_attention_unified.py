"""Attention without the score matrix on the GPU, forward and backward, against
the 64-bit form.

Bounds of the 2-norm: 16-bit types round the probabilities (and the backward
their gradients) to the type for the second product, errors of random sign of
at most u of each term, and the result once more: 2 u forward; 3 u for the
gradients, whose delta also comes from the rounded output.  float32: exponents
of about 20, 2^-24 * 20 of a probability, twice, and sums: 5e-6.
"""
from __future__ import annotations

import math

import pytest
import torch

import decoder_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _bounds(dt):
    return (5e-6, 8e-6) if dt == torch.float32 else (2 * ref.U[dt], 3 * ref.U[dt])


def _inputs(B, Tq, Tk, Hq, H, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * Tq + Tk + D)
    q, k, v, go = (torch.randn(s, generator=g).to(DEV, dtype)
                   for s in ((B, Tq, Hq, D), (B, Tk, H, D), (B, Tk, H, D), (B, Tq, Hq, D)))
    return q, k, v, go


def _check(q, k, v, go, mask=None, causal=False, scale=None):
    from axs.unified import axs_attention_unified

    print(f"q {tuple(q.shape)} k {tuple(k.shape)} {q.dtype} causal={causal}", flush=True)
    with torch.no_grad():
        alone = axs_attention_unified(q, k, v, mask, causal, scale)
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = axs_attention_unified(q, k, v, mask, causal, scale)
    grads = torch.autograd.grad(out, (q, k, v), go)
    want = ref.attention(q, k, v, go, mask, causal, scale)
    fwd, bwd = _bounds(q.dtype)
    assert torch.equal(alone, out.detach()) and out.dtype == q.dtype
    assert ref.rel(out.detach(), want[0]) <= fwd
    for name, x, y, of in zip("qkv", grads, want[1:], (q, k, v)):
        assert x.shape == of.shape and x.dtype == of.dtype
        # a gradient that is 0 (one key: dq, dk) is left with rounding of its terms
        assert ref.rel(x, y) <= bwd or float(y.norm()) <= 1e-9 * float(go.double().norm()) + 1e-300 and \
            float(x.double().norm()) <= bwd * float(go.double().norm() * k.detach().double().norm()), name
    return out, grads


SHAPES = [(1, 1, 1, 1, 1, 64), (2, 31, 33, 2, 2, 64), (1, 32, 64, 2, 1, 32), (1, 65, 65, 3, 1, 80), (2, 128, 129, 4, 2, 128),
          (1, 1, 200, 8, 2, 128), (1, 257, 100, 2, 2, 96), (1, 100, 257, 6, 2, 8), (3, 7, 5, 2, 1, 112), (1, 300, 300, 1, 1, 20)]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, causal, dtype):
    _check(*_inputs(*shape, dtype), causal=causal)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(1, 3, 2100, 2, 1, 64), (2, 1, 1030, 8, 2, 128), (1, 700, 333, 4, 1, 80), (1, 600, 600, 8, 8, 96)])
def test_split_axes(shape, causal, dtype):
    """Few rows against many keys (keys split), few keys against many queries (queries split); heads that divide by
    the chip's 8 dies."""
    _check(*_inputs(*shape, dtype), causal=causal)
    mask = torch.rand(shape[0], 1, 1, shape[2], generator=torch.Generator().manual_seed(1)) < 0.4
    mask[..., :300] = False     # whole tiles that nobody sees
    _check(*_inputs(*shape, dtype), mask=mask.to(DEV), causal=causal)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("D", [64, 72, 96, 128])
def test_many_workgroups(D, dtype):
    """The forms of larger problems: one group of waves a workgroup, and in the forward 256 queries a workgroup."""
    for causal in (False, True):
        _check(*_inputs(5, 190, 200, 32, 32, D, dtype), causal=causal)
    mask = torch.arange(200) < torch.tensor([[200], [50], [128], [1], [0]])
    _check(*_inputs(5, 190, 200, 32, 32, D, dtype), mask[:, None, None].to(DEV))


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(2, 128, 128, 4, 2, 64), (1, 127, 128, 3, 3, 64), (3, 128, 40, 2, 2, 64), (2, 97, 128, 8, 2, 48),
                                   (1, 129, 128, 2, 2, 64), (1, 128, 129, 2, 1, 64), (1, 33, 1, 2, 2, 32), (2, 160, 150, 2, 1, 64)])
def test_sequences_of_one_workgroup(shape, causal, dtype):
    """All of a head's tokens in one workgroup, which then makes all three gradients, and just past that: no mask, one
    by key, one by pair, and bad values where a causal mask or the mask hides them."""
    B, Tq, Tk, Hq, H, D = shape
    q, k, v, go = _inputs(*shape, dtype)
    _check(q, k, v, go, causal=causal)
    g = torch.Generator().manual_seed(2)
    by_key = (torch.rand(B, 1, 1, Tk, generator=g) < 0.6).to(DEV)
    by_key[0, ..., 32:64] = False
    _check(q, k, v, go, by_key, causal)
    by_pair = (torch.randn(B, Hq, Tq, Tk, generator=g) * 2).masked_fill(torch.rand(B, Hq, Tq, Tk, generator=g) < 0.3, -math.inf)
    _check(q, k, v, go, by_pair.to(DEV), causal)
    hidden = ~by_key[:, 0, 0].to(DEV)
    _, want = _check(q, k, v, go, by_key, causal)
    k[hidden] = math.nan
    v[hidden] = math.inf
    from axs.unified import axs_attention_unified
    qq, kk, vv = (x.detach().requires_grad_(True) for x in (q, k, v))
    got = torch.autograd.grad(axs_attention_unified(qq, kk, vv, by_key, causal), (qq, kk, vv), go)
    fwd, bwd = _bounds(dtype)
    for x, y, name in zip(got, want, "qkv"):
        if name != "q":     # rows of hidden keys: 0
            assert not x[hidden].any()
        assert ref.rel(x, y) <= 2 * bwd or float(y.double().norm()) == 0.0 == float(x.double().norm()), name


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("D", [1, 3, 33, 72, 127])
def test_odd_heads(D, dtype):
    _check(*_inputs(1, 70, 70, 2, 1, D, dtype), causal=True)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["padding", "full", "heads", "row", "empty", "none"])
def test_bool_masks(kind, causal, dtype):
    B, Tq, Tk, Hq, H, D = 2, 70, 90, 4, 2, 64
    q, k, v, go = _inputs(B, Tq, Tk, Hq, H, D, dtype)
    g = torch.Generator().manual_seed(5)
    if kind == "padding":
        mask = (torch.arange(Tk) < torch.tensor([[90], [33]]))[:, None, None, :]
    elif kind == "full":
        mask = torch.rand(B, Hq, Tq, Tk, generator=g) < 0.5
    elif kind == "heads":
        mask = (torch.rand(Hq, 1, Tk, generator=g) < 0.7)
    elif kind == "row":
        mask = torch.rand(Tk, generator=g) < 0.5
    elif kind == "empty":     # rows, a whole sequence, and the first tile of keys that see nothing
        mask = torch.rand(B, 1, Tq, Tk, generator=g) < 0.6
        mask[0, :, 5:9] = False
        mask[1] = False
        mask[0, :, 20, :64] = False
    else:
        mask = torch.zeros(1, 1, 1, Tk, dtype=torch.bool)
    out, grads = _check(q, k, v, go, mask.to(DEV), causal)
    dead = ~ref.seen(B, Hq, Tq, Tk, causal, mask)[0].any(-1).transpose(1, 2)
    assert not out[dead.to(DEV)].any() and not grads[0][dead.to(DEV)].any()


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("mask_dtype", ref.DTYPES)
def test_added_masks(mask_dtype, dtype):
    B, Tq, Tk, Hq, H, D = 2, 50, 70, 2, 1, 64
    q, k, v, go = _inputs(B, Tq, Tk, Hq, H, D, dtype)
    g = torch.Generator().manual_seed(6)
    add = torch.randn(B, 1, Tq, Tk, generator=g).to(mask_dtype)
    add[torch.rand(add.shape, generator=g) < 0.3] = -math.inf
    add[0, 0, 3] = -math.inf
    _check(q, k, v, go, add.to(DEV))
    _check(q, k, v, go, add.to(DEV)[:, :, :, ::2].repeat_interleave(2, 3), causal=True)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_the_lowest_value_as_a_mask(dtype):
    """Keys masked by the type's lowest value have no weight beside others; a row of them alone averages its
    keys (float32 and bfloat16: the scores vanish beside such a value)."""
    low = torch.finfo(torch.float32 if dtype == torch.float16 else dtype).min
    q, k, v, go = _inputs(1, 40, 70, 2, 2, 64, dtype)
    add = torch.zeros(1, 1, 40, 70, dtype=torch.float32 if dtype == torch.float16 else dtype)
    add[..., 35:] = low
    add[:, :, 7] = low
    from axs.unified import axs_attention_unified

    got = axs_attention_unified(q, k, v, add.to(DEV))
    want = ref.attention(q, k, v, mask=add)
    want[:, 7] = v.double().cpu().mean(1)
    assert ref.rel(got, want) <= _bounds(dtype)[0]


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_layouts_and_strides(dtype):
    B, T, Hq, H, D = 2, 60, 4, 2, 64
    q, k, v, go = _inputs(B, T, T, Hq, H, D, dtype)
    out, grads = _check(q, k, v, go, causal=True)
    # (B, H, T, D) in memory; one projection's rows of q, k and v; a row off the vector boundary; expanded batch
    by_head = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, go)]
    packed = torch.cat([x.flatten(2) for x in (q, k, v)], -1)
    parts = [x.unflatten(-1, (-1, D)) for x in packed.split([Hq * D, H * D, H * D], -1)]
    wide = [torch.nn.functional.pad(x, (1, 2))[..., 1:-2] for x in (q, k, v)]
    for a in (by_head, [*parts, go], [*wide, go]):
        o, g = _check(*a, causal=True)
        assert torch.equal(o, out) and all(torch.equal(x, y) for x, y in zip(g, grads))
    one = [x[:1].expand(B, -1, -1, -1) for x in (q, k, v)]
    _check(*one, go)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("Tk", [90, 2100])
def test_bad_values_where_nobody_looks(Tk, bad, dtype):
    """Infinities and NaN in keys and values that a query does not see have no part in its results, and queries that
    see nothing none in the keys'."""
    Tq = 70 if Tk == 90 else 6      # the longer keys are split over workgroups
    q, k, v, go = _inputs(2, Tq, Tk, 4, 2, 64, dtype)
    keep = torch.rand(2, 1, Tq, Tk, generator=torch.Generator().manual_seed(3)) < 0.7
    keep[..., 60:75] = False
    keep[:, :, 4] = False
    k[:, 60:70], v[0, 65:75, :, 5] = bad, bad
    q[:, 4], go[1, 4] = bad, bad
    _check(q, k, v, go, keep.to(DEV))
    pad = torch.ones(2, 1, 1, Tk, dtype=torch.bool)
    pad[..., 60:75] = False
    _check(*(torch.where(x.isfinite(), x, 0.5) if i in (0, 3) else x for i, x in enumerate((q, k, v, go))), pad.to(DEV))


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_bad_values_that_are_seen(dtype):
    """A NaN key or an infinite value reaches the rows that see it and no others."""
    from axs.unified import axs_attention_unified

    q, k, v, go = _inputs(1, 80, 80, 2, 2, 64, dtype)
    k[0, 50, 0], v[0, 40, 1, 7] = math.nan, math.inf
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    out = axs_attention_unified(*xs, causal=True)
    want, dq, dk, dv = ref.attention(q, k, v, go, causal=True)
    got = out.detach().double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert ref.rel(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0)) <= _bounds(dtype)[0]
    for x, y in zip(torch.autograd.grad(out, xs, go), (dq, dk, dv)):
        x = x.double().cpu()
        assert torch.equal(x.isfinite(), y.isfinite())
        assert ref.rel(torch.where(y.isfinite(), x, 0.0), torch.where(y.isfinite(), y, 0.0)) <= _bounds(dtype)[1]


def test_scale():
    q, k, v, go = _inputs(1, 40, 50, 2, 2, 64, torch.float32)
    for s in (1e-4, 0.5):
        _check(q, k, v, go, scale=s)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_large_scores(dtype):
    """Softmax close to one-hot, scores of about +-100."""
    q, k, v, go = _inputs(1, 64, 96, 2, 2, 64, dtype)
    q = q * 12
    from axs.unified import axs_attention_unified

    # 2^-24 * 150 of a probability
    assert ref.rel(axs_attention_unified(q, k, v), ref.attention(q, k, v)) <= 4 * _bounds(dtype)[0]


def test_zero_lengths():
    from axs.unified import axs_attention_unified

    for B, Tq, Tk, Hq, H in ((0, 4, 4, 2, 2), (1, 0, 4, 2, 1), (1, 4, 0, 2, 2), (2, 3, 3, 0, 0)):
        q = torch.ones(B, Tq, Hq, 64, device=DEV, requires_grad=True)
        k = torch.ones(B, Tk, H, 64, device=DEV, requires_grad=True)
        v = torch.ones(B, Tk, H, 64, device=DEV, requires_grad=True)
        out = axs_attention_unified(q, k, v)
        assert out.shape == q.shape and not out.any()
        for g in torch.autograd.grad(out.sum(), (q, k, v)):
            assert not g.any()


def test_gradients_against_differences():
    from axs.unified import axs_attention_unified

    q, k, v, go = _inputs(1, 37, 45, 4, 2, 40, torch.float32)
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(axs_attention_unified(*xs, causal=True), xs, go)
    g = torch.Generator().manual_seed(2)
    for i in range(3):
        d = torch.randn(xs[i].shape, generator=g).to(DEV)
        h = 1e-2   # truncation about h^2, rounding 2^-22 |f| / h
        with torch.no_grad():
            f = [float((axs_attention_unified(*[x + s * h * d if j == i else x for j, x in enumerate(xs)], causal=True)
                        .double() * go).sum()) for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - float((grads[i].double() * d).sum())) <= 3e-3 * float(grads[i].norm() * d.norm())


def test_same_bits_twice_and_on_another_stream():
    from axs.unified import axs_attention_unified

    q, k, v, go = (x.requires_grad_(True) for x in _inputs(2, 300, 300, 8, 2, 64, torch.bfloat16))

    def once():
        out = axs_attention_unified(q, k, v, causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), go))

    want = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = once()
    side.synchronize()
    for a, b, c in zip(want, once(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replays():
    from axs.unified import axs_attention_unified

    q, k, v, go = _inputs(2, 100, 100, 4, 2, 64, torch.float16)
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    torch.autograd.grad(axs_attention_unified(*xs, causal=True), xs, go)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = axs_attention_unified(*xs, causal=True)
        grads = torch.autograd.grad(out, xs, go)
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, *grads)]
        eager = axs_attention_unified(*xs, causal=True)
        for a, b in zip(got, (eager, *torch.autograd.grad(eager, xs, go))):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    from axs.unified import axs_attention_unified

    q, k, v, go = _inputs(2, 40, 70, 2, 1, 64, torch.bfloat16)
    step = 2 ** 31 + 64
    base = torch.empty(step + 2 * 70 * 64, device=DEV, dtype=torch.bfloat16)
    far = base.as_strided((2, 70, 1, 64), (step, 64, 64, 1))
    far.copy_(k)
    assert torch.equal(axs_attention_unified(q, far, v), axs_attention_unified(q, k, v))


def test_refusals():
    from axs.unified import axs_attention_unified as f

    q, k, v, _ = _inputs(2, 8, 8, 4, 2, 64, torch.float32)
    m = torch.ones(2, 1, 8, 8, dtype=torch.bool, device=DEV)
    for bad in (lambda: f(q[0], k, v), lambda: f(q.double(), k.double(), v.double()), lambda: f(q, k.half(), v),
                lambda: f(q, k[:1], v[:1]), lambda: f(q, k, v[:, :4]), lambda: f(q[:, :, :3], k, v),
                lambda: f(q, k[..., :32], v[..., :32]), lambda: f(q, k.cpu(), v), lambda: f(q, k, v, scale=0.0),
                lambda: f(q, k, v, scale=-1.0), lambda: f(q, k, v, scale=math.nan), lambda: f(q, k, v, m[..., :7]),
                lambda: f(q, k, v, m.long()), lambda: f(q, k, v, m.cpu()),
                lambda: f(q, k, v, torch.zeros(8, 8, device=DEV, requires_grad=True)),
                lambda: f(*[torch.zeros(1, 4, 1, 136, device=DEV)] * 3)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Tq,Tk", [(40, 33), (70, 40), (128, 127), (130, 40)])
def test_tokens_that_overlap_in_memory(Tq, Tk, causal, dtype):
    """Keys and values expanded over the tokens (one token's memory for all), and rows that overlap."""
    B, H, D = 2, 2, 64
    q, k, v, go = _inputs(B, Tq, Tk, H, H, D, dtype)
    _check(q, k[:, :1].expand(-1, Tk, -1, -1), v, go, causal=causal)
    # q, k: the same keys give every score of a row the same value, so tell them apart by overlapping windows
    step = 16
    mem = torch.randn(B, H, Tk * step + D, generator=torch.Generator().manual_seed(4)).to(DEV, dtype)
    near = mem.as_strided((B, Tk, H, D), (mem.stride(0), step, mem.stride(1), 1))
    _check(q, near, near, go, causal=causal)


def _low_rows(B, Hq, Tq, Tk, by_key, low):
    """An additive mask whose row 3 (by key: every row of sequence 1) carries `low` on all keys, and which of the
    (B, Tq) rows those are."""
    add = torch.zeros(B, 1, 1 if by_key else Tq, Tk)
    rows = torch.zeros(B, Tq, dtype=torch.bool)
    if by_key:
        add[1], rows[1] = low, True
    else:
        add[:, :, 3], rows[:, 3] = low, True
    return add, rows


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("low", [-1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("by_key", [False, True])
@pytest.mark.parametrize("B,Tq,Tk,Hq,H,D", [(2, 70, 100, 2, 1, 64), (2, 70, 100, 2, 1, 128), (2, 300, 200, 2, 2, 64),
                                            (2, 6, 2100, 2, 2, 64), (2, 700, 100, 4, 1, 96)])
def test_gradients_of_rows_of_large_finite_mask_values(B, Tq, Tk, Hq, H, D, by_key, low, dtype):
    """Beside such a value the scores vanish: the row's keys have equal probabilities, forward and backward.  The
    operands' sizes: one workgroup a head, several, the keys split, the queries split."""
    from axs.unified import axs_attention_unified

    q, k, v, go = _inputs(B, Tq, Tk, Hq, H, D, dtype)
    add, rows = _low_rows(B, Hq, Tq, Tk, by_key, low)
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    out = axs_attention_unified(*xs, add.to(DEV))
    got = (out.detach(), *torch.autograd.grad(out, xs, go))
    q, k, v, go = (x.detach().double().cpu() for x in (q, k, v, go))
    want = [torch.zeros_like(x) for x in (q, q, k, v)]
    for b in range(B):
        for h in range(Hq):
            g, scale = h // (Hq // H), 1 / math.sqrt(D)
            x = q[b, :, h] @ k[b, :, g].T * scale
            p = torch.softmax(torch.where(rows[b, :, None], 0.0, x), -1)
            dp = go[b, :, h] @ v[b, :, g].T
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            for i, y in enumerate((p @ v[b, :, g], ds @ k[b, :, g])):
                want[i][b, :, h] = y
            want[2][b, :, g] += ds.T @ q[b, :, h]
            want[3][b, :, g] += p.T @ go[b, :, h]
    fwd, bwd = _bounds(dtype)
    for i, (x, y) in enumerate(zip(got, want)):
        assert ref.rel(x, y) <= (bwd if i else fwd), "o dq dk dv".split()[i]
        if i < 2:    # the rows by themselves
            assert ref.rel(x[rows.to(DEV)], y[rows]) <= (bwd if i else fwd), "o dq".split()[i]


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_one_sequence_or_token_of_an_unaligned_batch(dtype):
    """A dim of one element may have any stride: it is never walked."""
    q, k, v, go = _inputs(1, 1, 5, 2, 2, 64, dtype)
    want, grads = _check(q, k, v, go)

    def odd(x, dim):    # x with a stride of 1 along a dim of one element
        strides = list(x.stride())
        strides[dim] = 1
        return x.as_strided(x.shape, strides)

    for qq, kk, vv, gg in ((odd(q, 0), odd(k, 0), odd(v, 0), odd(go, 0)), (odd(q, 1), k, v, odd(go, 1))):
        out, got = _check(qq, kk, vv, gg)
        assert torch.equal(out, want) and all(torch.equal(x, y) for x, y in zip(got, grads))
    batch = torch.randn(2, 5 * 2 * 64 + 1, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    one = batch[:, :-1].unflatten(-1, (5, 2, 64))[:1]
    _check(q, one, one, go)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Tq,Tk,D", [(1024, 1024, 64), (4096, 4096, 64), (128, 128, 64), (300, 2048, 80), (600, 600, 128)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4])
def test_small_float16_gradients(size, Tq, Tk, D, causal):
    """float16 gradients from small ones of the output: the error is that of the products' operands, 3 u of the
    gradient, and the result's own rounding, half a step of float16 (2^-24 below 2^-14)."""
    from axs.unified import axs_attention_unified

    q, k, v, go = _inputs(1, Tq, Tk, 1, 1, D, torch.float16)
    go = (go.float() * size).half()
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    got = torch.autograd.grad(axs_attention_unified(*xs, causal=causal), xs, go)
    for name, x, y in zip("qkv", got, ref.attention(q, k, v, go, causal=causal)[1:]):
        error = float((x.double().cpu() - y).norm())
        assert error <= 3 * ref.U[torch.float16] * float(y.norm()) + 2.0 ** -25 * math.sqrt(y.numel()), name


def test_float16_gradients_of_large_ones_and_of_long_rows():
    """Score gradients past float16's largest value behind small keys and queries; probabilities far below its
    smallest normal one."""
    from axs.unified import axs_attention_unified

    for Tq, Tk, D in ((100, 8, 64), (200, 9, 64), (130, 140, 128)):
        q, k, v, go = _inputs(1, Tq, Tk, 2, 1, D, torch.float16)
        _check(q * 0.01, k * 0.01, v * 300, go * 300)
    q, k, v, go = _inputs(1, 48, 200000, 1, 1, 32, torch.float16)
    xs = [x.requires_grad_(True) for x in (q, k, v)]
    got = torch.autograd.grad(axs_attention_unified(*xs), xs, go)
    for name, x, y in zip("qkv", got, ref.attention(q, k, v, go)[1:]):
        error = float((x.double().cpu() - y).norm())
        assert error <= 3 * ref.U[torch.float16] * float(y.norm()) + 2.0 ** -25 * math.sqrt(y.numel()), name
