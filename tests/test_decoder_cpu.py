"""The decoder's operators without a GPU: host tensors and bad arguments are
refused, the C entries check before they touch a device, the rotary table."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from axs import _lib


def test_host_tensors_raise_cuda_error():
    import axs.unified as axu

    x = torch.zeros(1, 4, 2, 32)
    n = torch.zeros(1, dtype=torch.int64)
    cache = axu.AXSKVCacheUnified.empty(1, 2, 32, 64, device="cpu")
    assert cache.max_tokens == 64 and cache.v_codes.shape == (1, 2, 2, 32, 32)
    for call in (lambda: axu.axs_rotary_unified(x, x, axu.rotary_table(32, 8)),
                 lambda: axu.axs_attention_unified(x, x, x),
                 lambda: axu.axs_cache_append_unified(cache, x, x, n),
                 lambda: axu.axs_cache_read_unified(cache, n, 4),
                 lambda: axu.axs_cache_attention_unified(x, cache, n),
                 lambda: axu.axs_distillation_loss_unified(x[0, 0], x[0, 0, :, :4], torch.zeros(2, 4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_rotary_table():
    from axs.unified import rotary_table

    t = rotary_table(8, 50, base=100.0)
    i = torch.arange(4, dtype=torch.float64)
    angle = torch.arange(50, dtype=torch.float64)[:, None] * 100.0 ** (-i / 4)
    assert torch.equal(t, torch.cat([angle.cos(), angle.sin()], 1).float())
    lin = rotary_table(8, 50, base=100.0, scaling="linear", factor=4.0)
    assert torch.allclose(lin[::4], t[:13], atol=1e-6)
    # the lowest frequency is stretched by the factor, the highest stays
    ntk = rotary_table(8, 50, base=100.0, scaling="base", factor=4.0)
    assert torch.equal(ntk[:, 0], t[:, 0]) and torch.allclose(ntk[::4, 3], t[:13, 3], atol=1e-5)
    parts = rotary_table(128, 50, scaling="parts", factor=4.0, original_positions=4096)
    gain = 0.1 * math.log(4.0) + 1.0
    plain = rotary_table(128, 50)
    assert torch.allclose(parts[:, 0], plain[:, 0] * gain, atol=1e-6)
    assert torch.allclose(parts[::4, 63], plain[:13, 63] * gain, atol=1e-6)
    assert rotary_table(0, 3).shape == (3, 0)
    for bad in ({"rotary_dim": 7}, {"max_positions": 0}, {"base": 0.5}, {"factor": 0.5}, {"scaling": "other"},
                {"scaling": "parts"}):
        with pytest.raises(ValueError):
            rotary_table(**({"rotary_dim": 8, "max_positions": 4} | bad))


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_c_entries_check_their_arguments():
    L = _lib.lib()
    st = ctypes.cast(_i64(256, 64, 64, 1), ctypes.c_void_p)
    p, odd = 4096, 4098   # never read: every call below is refused, or has nothing to do
    fwd = L.axs6_attention_forward
    good = [p, p, p, 0, 1, 4, 4, 2, 1, 64, st, st, st, None, 0, None, 0, 0.1, p, p, None, 0, None]

    def call(fn, args, **changes):
        a = list(args)
        for i, x in changes.items():
            a[int(i[1:])] = x
        return fn(*a)

    for change, rc in (({"a3": 9}, 1), ({"a7": 3, "a8": 2}, 1), ({"a9": 136}, 2), ({"a9": 63}, 2), ({"a17": 0.0}, 1),
                       ({"a17": math.inf}, 1), ({"a0": None}, 1), ({"a1": odd}, 1), ({"a18": None}, 1), ({"a4": -1}, 1),
                       ({"a13": p}, 1), ({"a13": p, "a14": 7, "a15": st}, 1), ({"a5": 1 << 31}, 2), ({"a5": 0}, 0),
                       ({"a10": ctypes.cast(_i64(256, 63, 64), ctypes.c_void_p)}, 1),
                       ({"a11": ctypes.cast(_i64(256, 1 << 22, 64), ctypes.c_void_p)}, 2)):
        assert call(fwd, good, **change) == rc, change
        assert rc == 0 or L.axs6_last_error()
    bwd = [p, p, p, p, p, p, 0, 1, 4, 4, 2, 1, 64, st, st, st, st, None, 0, None, 0, 0.1, p, p, p, p, p, 1 << 20, None]
    for change, rc in (({"a6": 5}, 1), ({"a0": None}, 1), ({"a5": None}, 1), ({"a23": odd}, 1), ({"a22": None}, 1),
                       ({"a7": 0}, 0), ({"a8": 1 << 14, "a9": 1 << 14}, 1)):
        assert call(L.axs6_attention_backward, bwd, **change) == rc, change
    rot = [p, p, p, p, 0, 1, 4, 2, 1, 64, 32, st, st, p, 10, None, 0, 0, 0, 0, None]
    for change, rc in (({"a10": 31}, 1), ({"a10": 66}, 1), ({"a9": 600}, 2), ({"a13": None}, 1), ({"a2": None}, 1),
                       ({"a0": odd + 1}, 1), ({"a6": 0}, 0), ({"a4": 3}, 1)):
        assert call(L.axs6_rotary, rot, **change) == rc, change
    app = [p, p, 0, 1, 4, 1, 64, st, st, p, 4, p, p, p, p, p, p, None]
    for change, rc in (({"a6": 40}, 2), ({"a6": 272}, 2), ({"a9": None}, 1), ({"a11": odd}, 1), ({"a4": 0}, 0),
                       ({"a2": 4}, 1), ({"a15": odd}, 1), ({"a10": 1 << 26}, 1), ({"a10": 0}, 0)):
        assert call(L.axs6_kv_append, app, **change) == rc, change
    read = [p, p, p, p, 1, 1, 64, 4, p, 4, p, p, None]
    for change, rc in (({"a8": None}, 1), ({"a9": -1}, 2), ({"a10": odd}, 1), ({"a9": 0}, 0), ({"a0": None}, 1)):
        assert call(L.axs6_kv_read, read, **change) == rc, change
    att = [p, 0, 1, 1, 4, 2, 64, st, p, p, p, p, 4, p, 0.1, p, None, 0, None]
    for change, rc in (({"a4": 3}, 1), ({"a12": 0}, 1), ({"a14": math.nan}, 1), ({"a12": 4096}, 1), ({"a3": 0}, 0),
                       ({"a15": None}, 1), ({"a1": 3}, 1)):
        assert call(L.axs6_kv_attention, att, **change) == rc, change
    assert call(fwd, good, a6=8192) == 1   # split keys need a workspace
    assert L.axs6_attention_forward_workspace(1, 4, 8192, 2, 64) > 0
    assert L.axs6_attention_forward_workspace(1, 4, 64, 2, 64) == 0
    assert L.axs6_attention_backward_workspace(0, 4, 64, 2, 1, 64, 1) == 0
    need = L.axs6_kv_attention_workspace(1, 1, 4, 2, 64, 4096)
    assert need > 0 and L.axs6_kv_attention_workspace(0, 1, 4, 2, 64, 4096) == 0
    dis = [p, 0, 100, 4, 100, p, p, 8, 1.0, None, 1, p, p, p, p, None]
    for change, rc in (({"a1": 8}, 1), ({"a2": 99}, 1), ({"a8": 0.0}, 1), ({"a8": math.nan}, 1), ({"a5": None}, 1),
                       ({"a11": None}, 1), ({"a14": None}, 1), ({"a0": odd}, 1)):
        assert call(L.axs6_distill_forward, dis, **change) == rc, change
    dis = [p, 0, 100, 4, 100, p, p, 8, 1.0, None, p, p, 0, p, p, None]
    for change, rc in (({"a10": None}, 1), ({"a11": None}, 1), ({"a14": None}, 1), ({"a3": 0}, 0)):
        assert call(L.axs6_distill_backward, dis, **change) == rc, change


@pytest.mark.parametrize("rotary_dim,original,base", [(128, 4096, 1e4), (128, 131072, 1e4), (128, 65536, 1e4), (64, 32768, 1e6),
                                                      (80, 300, 1e4), (32, 6, 1e4), (128, 2, 1e4)])
def test_rotary_table_by_parts(rotary_dim, original, base):
    """By wavelength: 32 turns or more within the original positions stay, one at most is divided by the factor, a
    linear ramp over the index between, also where that ends past the last index."""
    from axs.unified import rotary_table

    factor, n = 4.0, rotary_dim // 2
    t = rotary_table(rotary_dim, 2, base=base, scaling="parts", factor=factor, original_positions=original).double()
    got = torch.atan2(t[1, n:], t[1, :n])               # the frequencies: angles of position 1
    i = torch.arange(n, dtype=torch.float64)
    whole = base ** (-i / n)
    turns = whole * original / (2 * math.pi)
    kept = 1 - (got / whole - 1 / factor) / (1 - 1 / factor)    # 0: as it was, 1: divided in full
    assert kept[turns <= 1].sub(1).abs().le(1e-5).all() and kept[turns >= 32].abs().le(1e-5).all()
    # between: a line over the index from the last that stays to the first that is divided in full
    at = lambda k: n * math.log(original / (2 * math.pi * k)) / math.log(base)
    low, high = max(math.floor(at(32)), 0), math.ceil(at(1))
    between = (i > low) & (i < high)
    assert (kept - (i - low) / max(high - low, 1))[between].abs().le(1e-5).all()
    assert not ((kept > 1 - 1e-5) & (turns > 1) & (i < high)).any()


def test_row_statistics_are_aligned():
    L = _lib.lib()
    st = ctypes.cast(_i64(256, 64, 64, 1), ctypes.c_void_p)
    p, half = 4096, 4100
    assert L.axs6_attention_forward(p, p, p, 0, 1, 4, 4, 2, 1, 64, st, st, st, None, 0, None, 0, 0.1, p, half, None, 0, None) == 1
    assert L.axs6_attention_backward(p, p, p, p, p, half, 0, 1, 4, 4, 2, 1, 64, st, st, st, st, None, 0, None, 0, 0.1, p, p, p,
                                     p, p, 1 << 20, None) == 1


@pytest.mark.parametrize("B,Tq,Hq,H,D", [(1, 4096, 32, 8, 128), (1, 16384, 32, 8, 128), (4, 512, 32, 8, 128), (1, 100, 8, 1, 256),
                                         (64, 1, 64, 8, 128), (1, 1, 32, 8, 128), (8, 5, 64, 8, 128), (1, 1 << 20, 8, 8, 64)])
@pytest.mark.parametrize("capacity", [512, 16384, 131072, 1 << 20])
def test_cache_attention_workspace_stays_small(B, Tq, Hq, H, D, capacity):
    """Partial sums of a long prompt do not grow with the cache's capacity."""
    rows = B * Tq * Hq * (D + 2) * 4        # bytes of one split's
    need = _lib.lib().axs6_kv_attention_workspace(B, Tq, Hq, H, D, capacity // 32)
    assert need % rows == 0 and need <= 64 << 20
