"""The decoder's operators together: the self-attention module against its parts,
the example's training from a teacher, and its answers from the 8-bit cache
against the whole-sequence forward."""
from __future__ import annotations

import importlib.util
import os
import sys

import pytest
import torch

import decoder_ref as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _example():
    spec = importlib.util.spec_from_file_location("distill_decoder",
                                                  os.path.join(ROOT, "axs-6_amd", "examples", "distill_decoder.py"))
    m = sys.modules[spec.name] = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("kv_heads", [None, 2, 1])
def test_self_attention_is_its_parts(kv_heads):
    import axs.unified as axu

    torch.manual_seed(0)
    m = axu.AXSCausalSelfAttentionUnified(128, 4, kv_heads).to(DEV)
    table = axu.rotary_table(32, 64, device=DEV)
    x = torch.randn(2, 40, 128, device=DEV, requires_grad=True)
    y = m(x, table)
    q, k, v = (p(x).unflatten(-1, (-1, 32)) for p in (m.q_proj, m.k_proj, m.v_proj))
    q, k = axu.axs_rotary_unified(q, k, table)
    parts = m.out_proj(axu.axs_attention_unified(q, k, v, causal=True).flatten(2))
    assert torch.equal(y, parts)
    y.sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters()) and x.grad.isfinite().all()


def test_decode_follows_the_whole_forward():
    """Float32: the cache's 8 bits leave errors of at most 1/254 of a block's largest value in keys and values."""
    import axs.unified as axu

    torch.manual_seed(0)
    m = axu.AXSCausalSelfAttentionUnified(128, 4, 2).to(DEV)
    table = axu.rotary_table(32, 128, device=DEV)
    x = torch.randn(3, 70, 128, device=DEV)
    with torch.no_grad():
        want = m(x, table)
    cache = m.new_cache(3, 70, device=DEV)
    got = [m.decode(x[:, :37], table, cache, torch.zeros(3, dtype=torch.int64, device=DEV))]
    for t in range(37, 70):
        got.append(m.decode(x[:, t:t + 1], table, cache, torch.full((3,), t, dtype=torch.int64, device=DEV)))
    # scores and values each off by about 1/254 of a largest value of 3 deviations, averaged over values: 3%
    assert ref.rel(torch.cat(got, 1), want) <= 0.03


def test_example_learns_and_answers():
    ex = _example()
    c = ex.Config(batch=16, context=64)
    teacher = ex.train_teacher(c, 150, DEV)
    student, losses = ex.distill(c, teacher, 150, DEV)
    assert losses[-1] < 0.5 * losses[0]
    prompt = ex.sequences(c, torch.Generator().manual_seed(9), DEV)[:, :24]
    out = student.generate(prompt, 8)
    assert out.shape == (16, 32) and torch.equal(out[:, :24], prompt)
    # the answers are the whole forward's, but where two classes are nearly equal
    with torch.no_grad():
        whole = student(out[:, :-1])[:, 23:]
    top = whole.topk(2, -1).values
    sure = top[..., 0] - top[..., 1] > 0.1 * whole.std()
    assert torch.equal(whole.argmax(-1)[sure], out[:, 24:][sure])


@pytest.mark.parametrize("setting", [{"quantize_input": False}, {"quantize_grad": False}, {"block_size": 16}])
@pytest.mark.parametrize("which", ["q_proj", "k_proj", "v_proj"])
def test_each_projection_keeps_its_settings(which, setting):
    """Settings of one projection, or a projection of another type, hold in forward, backward and decode."""
    import axs.unified as axu

    torch.manual_seed(0)
    m = axu.AXSCausalSelfAttentionUnified(128, 4, 2).to(DEV)
    for name, value in setting.items():
        setattr(getattr(m, which), name, value)
    _is_its_parts(m)


@pytest.mark.parametrize("which", ["q_proj", "k_proj", "v_proj"])
def test_projections_of_another_type(which):
    import axs.unified as axu

    torch.manual_seed(0)
    m = axu.AXSCausalSelfAttentionUnified(128, 4, 2).to(DEV)
    p = getattr(m, which)
    setattr(m, which, torch.nn.Linear(p.in_features, p.out_features).to(DEV))
    _is_its_parts(m)
    m = axu.AXSCausalSelfAttentionUnified(128, 4, 2, block_size=16).to(DEV)
    _is_its_parts(m, gradients=False)    # grouped: rounded by other random numbers


def _is_its_parts(m, gradients=True):
    import axs.unified as axu

    table = axu.rotary_table(32, 64, device=DEV)
    x = torch.randn(2, 40, 128, device=DEV, requires_grad=True)
    go = torch.randn(2, 40, 128, device=DEV)

    def heads():
        return (p(x).unflatten(-1, (-1, 32)) for p in (m.q_proj, m.k_proj, m.v_proj))

    y = m(x, table)
    params = list(m.parameters())
    torch.manual_seed(5)    # of the gradients' stochastic rounding
    got = torch.autograd.grad(y, [x, *params], go)
    q, k, v = heads()
    q, k = axu.axs_rotary_unified(q, k, table)
    parts = m.out_proj(axu.axs_attention_unified(q, k, v, causal=True).flatten(2))
    assert torch.equal(y, parts)
    torch.manual_seed(5)
    for a, b in zip(got, torch.autograd.grad(parts, [x, *params], go)):
        assert not gradients or ref.rel(a, b) <= 1e-5
    with torch.no_grad():
        cache, other = (m.new_cache(2, 40, device=DEV) for _ in range(2))
        starts = torch.zeros(2, dtype=torch.int64, device=DEV)
        out = m.decode(x, table, cache, starts)
        q, k, v = heads()
        q, k = axu.axs_rotary_unified(q, k, table)
        axu.axs_cache_append_unified(other, k, v, starts)
        want = m.out_proj(axu.axs_cache_attention_unified(q, other, starts + 40).flatten(2))
    assert torch.equal(out, want)


def test_forward_mode_tangents_raise():
    """The operators have no forward-mode derivative: a tangent raises, as in the linear, and is never dropped."""
    import torch.autograd.forward_ad as fwd
    from axs.unified import axs_attention_unified, axs_distillation_loss_unified, axs_rotary_unified, rotary_table

    x = torch.randn(1, 8, 2, 16, device=DEV)
    table = rotary_table(16, 8, device=DEV)
    z, t, i = torch.randn(4, 10, device=DEV), torch.randn(4, 2, device=DEV), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: axs_rotary_unified(d, x, table), lambda: axs_rotary_unified(x, d, table),
                     lambda: axs_rotary_unified(d, None, table), lambda: axs_attention_unified(d, x, x),
                     lambda: axs_attention_unified(x, d, x), lambda: axs_attention_unified(x, x, d),
                     lambda: axs_distillation_loss_unified(fwd.make_dual(z, torch.ones_like(z)), t, i)):
            with pytest.raises(RuntimeError, match="jvp"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                call()
        # without a tangent nothing changes
        assert axs_rotary_unified(x, x, table)[0].shape == x.shape and axs_attention_unified(x, x, x).shape == x.shape
