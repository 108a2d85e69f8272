"""Rotary positions on the GPU against the 64-bit form.

A result is a sum of two products in float32, rounded once to the type:
|error| <= u |y| + 3 * 2^-24 (|a| + |b|), at most (2 u + 6 * 2^-24) in the norm.
"""
from __future__ import annotations

import pytest
import torch

import decoder_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _bound(dt):
    return (2 * ref.U[dt] if dt != torch.float32 else 0) + 6 * ref.U[torch.float32]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R", [
    (1, 1, 1, 1, 2, 2), (2, 1, 32, 8, 128, 128), (3, 37, 4, 2, 64, 32), (1, 5, 3, 1, 7, 4), (2, 9, 5, 5, 80, 80),
    (1, 300, 6, 2, 96, 48), (2, 17, 4, 4, 40, 8), (1, 3, 2, 1, 512, 512), (2, 4, 2, 2, 33, 0), (5, 129, 8, 2, 128, 16), (2, 31, 5, 1, 80, 40), (1, 50, 2, 2, 36, 24),
])
def test_rotation_and_gradient(B, T, Hq, Hkv, D, R, interleaved, dtype):
    from axs.unified import axs_rotary_unified, rotary_table

    g = torch.Generator().manual_seed(B * 1000 + T)
    table = rotary_table(R, 500, device=DEV)
    q = torch.randn(B, T, Hq, D, generator=g).to(DEV, dtype).requires_grad_(True)
    k = torch.randn(B, T, Hkv, D, generator=g).to(DEV, dtype).requires_grad_(True)
    pos = torch.randint(0, 500, (B, T), generator=g)
    gq, gk = (torch.randn(x.shape, generator=g).to(DEV, dtype) for x in (q, k))
    yq, yk = axs_rotary_unified(q, k, table, pos.to(DEV), interleaved)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    assert yq.dtype == dtype and yq.is_contiguous()
    for got, x, inv in ((yq, q, False), (yk, k, False), (dq, gq, True), (dk, gk, True)):
        assert ref.rel(got.detach(), ref.rotate(x.detach(), table, pos, interleaved, inv)) <= _bound(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_layouts_and_one_operand(dtype):
    from axs.unified import axs_rotary_unified, rotary_table

    g = torch.Generator().manual_seed(3)
    table = rotary_table(32, 64, device=DEV)
    qkv = torch.randn(2, 12, 3 * 4 * 32 + 1, generator=g).to(DEV, dtype)
    q = qkv[..., 1:1 + 128].unflatten(-1, (4, 32))        # rows off any vector boundary
    k = torch.randn(2, 4, 12, 32, generator=g).to(DEV, dtype).transpose(1, 2)   # (B, H, T, D) in memory
    order = torch.arange(12)
    y0, z0 = axs_rotary_unified(q, k, table)
    for pos in (order, order.int(), order[None], order.expand(2, 12)):
        y, z = axs_rotary_unified(q, k, table, pos.to(DEV))
        assert torch.equal(y, y0) and torch.equal(z, z0)
    assert ref.rel(y0, ref.rotate(q, table, order, False)) <= _bound(dtype)
    assert ref.rel(z0, ref.rotate(k, table, order, False)) <= _bound(dtype)
    y, none = axs_rotary_unified(q, None, table)
    assert none is None and torch.equal(y, y0)
    x = k.detach().requires_grad_(True)                   # a gradient for the keys alone
    dk, = torch.autograd.grad(axs_rotary_unified(q, x, table)[1].sum(), x)
    assert ref.rel(dk, ref.rotate(torch.ones_like(k), table, order, False, True)) <= _bound(dtype)


def test_outside_the_table_and_empty():
    from axs.unified import axs_rotary_unified, rotary_table

    table = rotary_table(8, 10, device=DEV)
    q = torch.ones(1, 4, 1, 16, device=DEV)
    y, _ = axs_rotary_unified(q, None, table, torch.tensor([0, -1, 10, 9], device=DEV))
    assert y[0, (1, 2), :, :8].isnan().all() and not y[0, (0, 3)].isnan().any()
    assert torch.equal(y[..., 8:], q[..., 8:])
    for shape in ((0, 4, 1, 16), (1, 0, 1, 16), (1, 4, 0, 16)):
        assert axs_rotary_unified(torch.empty(shape, device=DEV), None, table)[0].shape == shape


def test_refusals():
    from axs.unified import axs_rotary_unified, rotary_table

    t, q = rotary_table(8, 10, device=DEV), torch.zeros(1, 4, 1, 16, device=DEV)
    for bad in (lambda: axs_rotary_unified(q[0], None, t), lambda: axs_rotary_unified(q.double(), None, t),
                lambda: axs_rotary_unified(q, q.half(), t), lambda: axs_rotary_unified(q, q[:, :2], t),
                lambda: axs_rotary_unified(q, None, t.double()), lambda: axs_rotary_unified(q[..., :4], None, t),
                lambda: axs_rotary_unified(q, None, t[:, :3]), lambda: axs_rotary_unified(q, None, t[:2]),
                lambda: axs_rotary_unified(q, None, t, torch.zeros(3, dtype=torch.int64, device=DEV)),
                lambda: axs_rotary_unified(q, None, t, torch.zeros(4, device=DEV)),
                lambda: axs_rotary_unified(q, None, t, torch.zeros(4, dtype=torch.int64)),
                lambda: axs_rotary_unified(torch.zeros(1, 1, 1, 514, device=DEV), None, t)):
        with pytest.raises(RuntimeError):
            bad()
