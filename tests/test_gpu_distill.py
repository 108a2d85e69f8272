"""The distillation loss on the GPU against the 64-bit form.

float32 exponentials of exponents up to about 40 in size and sums over V
classes: 2^-24 (40 + 8) < 3e-6 of the loss's terms and of a probability; the
loss is a difference of terms a few times its size, so 2e-5 of it.  Gradients
add their type's unit roundoff.
"""
from __future__ import annotations

import math

import pytest
import torch

import decoder_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _bound(dt):
    return (ref.U[dt] if dt != torch.float32 else 0) + 3e-6


def _case(N, V, K, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed + N + V + K)
    z = (torch.randn(N, V, generator=g) * scale).to(DEV, dtype).requires_grad_(True)
    values = (torch.randn(N, K, generator=g) * scale).to(DEV)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]) if N else torch.empty(0, K, dtype=torch.long)
    w = (torch.rand(N, generator=g) * (torch.rand(N, generator=g) < 0.8)).to(DEV)
    return z, values, idx.to(DEV), w


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N,V,K,T", [(1, 1, 1, 1.0), (3, 7, 4, 0.5), (5, 1000, 8, 2.0), (2, 4096, 64, 1.0),
                                     (4, 511, 511, 4.0), (1, 50001, 20, 1.5), (9, 2056, 1, 3.0)])
def test_loss_and_gradient(N, V, K, T, reduction, dtype):
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, w = _case(N, V, K, dtype)
    loss = axs_distillation_loss_unified(z, values, idx, T, w, reduction)
    grad, = torch.autograd.grad(loss.sum(), z)
    want, dz = ref.distill(z, values, idx, T, w, reduction)
    assert loss.dtype == torch.float32 and grad.dtype == dtype
    # a loss near 0 is a difference of terms of about T^2 log V
    assert float((loss.detach().double().cpu() - want).abs().max()) <= 2e-5 * float(want.abs().max()) + 3e-6 * T * T * 12
    assert ref.rel(grad, dz) <= _bound(dtype) or float(dz.norm()) < 1e-6 * T * max(N, 1)


def test_left_out_repeated_and_bad_entries():
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, _ = _case(6, 300, 5, torch.float32)
    idx[0, 2:] = -1            # fewer entries
    idx[1] = -7                # none at all: no loss, no gradient
    idx[2, 1:4] = idx[2, 0]    # one class four times
    idx[3, 2] = 300            # past the classes
    values[4, 1] = -math.inf   # a probability of 0
    with torch.no_grad():
        z[5, :200] = -math.inf
    idx[5] = torch.arange(200, 205, device=DEV)
    for reduction in ("none", "sum"):
        loss = axs_distillation_loss_unified(z, values, idx, 1.0, None, reduction)
        grad, = torch.autograd.grad(loss.sum(), z)
        want, dz = ref.distill(z, values, idx, 1.0, None, reduction)
        assert torch.equal(loss.isnan().cpu(), want.isnan())
        ok = [0, 1, 2, 4, 5]
        assert ref.rel(grad[ok], dz[ok]) <= 3e-6 and grad[3].isnan().all()
        if reduction == "none":
            assert ref.rel(loss[ok].detach(), want[ok]) <= 2e-5
            assert loss[1] == 0


def test_weights_of_zero_hide_a_row_and_a_sum_of_zero():
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, _ = _case(3, 64, 4, torch.float32)
    with torch.no_grad():
        z[1] = math.nan
    w = torch.tensor([1.0, 0.0, 2.0], device=DEV)
    loss = axs_distillation_loss_unified(z, values, idx, 1.0, w)
    grad, = torch.autograd.grad(loss, z)
    keep = [0, 2]
    want, dz = ref.distill(z[keep], values[keep], idx[keep], 1.0, w[keep])
    assert abs(float(loss) - float(want)) <= 2e-5 * abs(float(want))
    assert ref.rel(grad[keep], dz) <= 3e-6 and not grad[1].any()
    none = axs_distillation_loss_unified(z, values, idx, 1.0, torch.zeros(3, device=DEV))
    assert float(none) == 0 and not torch.autograd.grad(none, z)[0].any()


def test_strided_rows_batch_dims_and_int32():
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, w = _case(6, 100, 4, torch.bfloat16)
    wide = torch.zeros(6, 131, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:103] = z.detach()
    view = wide[:, 3:103].requires_grad_(True)
    a = axs_distillation_loss_unified(z, values, idx, 2.0, w)
    b = axs_distillation_loss_unified(view, values, idx.int(), 2.0, w)
    c = axs_distillation_loss_unified(z.view(2, 3, 100), values.view(2, 3, 4), idx.view(2, 3, 4), 2.0, w.view(2, 3))
    assert abs(float(a - b)) <= 1e-6 * float(a) and torch.equal(a, c)
    assert torch.equal(torch.autograd.grad(a, z)[0], torch.autograd.grad(c, z)[0])


def test_gradient_against_differences():
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, w = _case(4, 97, 6, torch.float32)
    g, = torch.autograd.grad(axs_distillation_loss_unified(z, values, idx, 1.5, w, "sum"), z)
    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    h = 1e-2   # truncation h^2 |f'''| ~ 1e-4, rounding 2^-22 |f| / h ~ 1e-4
    with torch.no_grad():
        up, down = (axs_distillation_loss_unified(z + s * h * d, values, idx, 1.5, w, "sum") for s in (1, -1))
    slope = float(up - down) / (2 * h)
    assert abs(slope - float((g * d).sum())) <= 3e-3 * float(g.norm() * d.norm())


def test_loss_scale_reaches_small_gradients():
    """float16: the upstream factor multiplies before the one rounding."""
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, _ = _case(2, 40000, 4, torch.float16, scale=1.0)
    loss = axs_distillation_loss_unified(z, values, idx, 1.0)
    grad, = torch.autograd.grad(loss * 65536.0, z)
    _, dz = ref.distill(z, values, idx, 1.0)
    assert ref.rel(grad, dz * 65536.0) <= _bound(torch.float16)


def test_refusals():
    from axs.unified import axs_distillation_loss_unified as f

    z, v, i, w = _case(3, 16, 4, torch.float32)
    for bad in (lambda: f(z.double(), v, i), lambda: f(z, v[:2], i[:2]), lambda: f(z, v, i[:, :2]),
                lambda: f(z, v, i.float()), lambda: f(z, v, i, 0.0), lambda: f(z, v, i, -1.0),
                lambda: f(z, v, i, math.inf), lambda: f(z, v, i, 1.0, w[:2]), lambda: f(z, v.cpu(), i),
                lambda: f(z, v, i.cpu()), lambda: f(z, v.clone().requires_grad_(True), i)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        f(z, v, i, 1.0, None, "average")


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("batch", [(), (6,), (2, 3), (1, 6), (2, 1, 3)])
def test_batch_dims_and_reductions(batch, reduction, dtype):
    from axs.unified import axs_distillation_loss_unified

    z, values, idx, w = _case(max(1, math.prod(batch)), 100, 4, dtype)
    w[0] = 0.5
    z = z.detach().view(*batch, 100).requires_grad_(True)
    values, idx, w = values.view(*batch, 4), idx.view(*batch, 4), w.view(batch)
    loss = axs_distillation_loss_unified(z, values, idx, 2.0, w, reduction)
    assert loss.shape == (batch if reduction == "none" else ())
    grad, = torch.autograd.grad(loss.sum(), z)
    want, dz = ref.distill(z, values, idx, 2.0, w, reduction)
    want = want.view(loss.shape)
    assert float((loss.detach().double().cpu() - want).abs().max()) <= 2e-5 * float(want.abs().max()) + 3e-6 * 4 * 12
    assert grad.shape == z.shape and ref.rel(grad.reshape(-1, 100), dz) <= _bound(dtype)
