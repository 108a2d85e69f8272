"""Beam search's operators without a GPU: host tensors and bad arguments are refused,
the C entries check before they touch a device."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from axs import _lib


def test_host_tensors_raise_cuda_error():
    import axs.unified as axu

    n = torch.zeros(2, dtype=torch.int64)
    cache = axu.AXSKVCacheUnified.empty(2, 2, 32, 64, device="cpu")
    for call in (lambda: axu.axs_beam_select_unified(torch.zeros(1, 2, 5), torch.zeros(1, 2)),
                 lambda: axu.axs_cache_copy_unified(cache, n, n),
                 lambda: axu.axs_cache_shared_attention_unified(torch.zeros(2, 1, 2, 32), cache, n, cache, n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def _i64(*v):
    return ctypes.cast((ctypes.c_int64 * len(v))(*v), ctypes.c_void_p)


def _call(fn, args, **changes):
    a = list(args)
    for i, x in changes.items():
        a[int(i[1:])] = x
    return fn(*a)


def test_select_checks_its_arguments():
    L = _lib.lib()
    p, odd = 4096, 4098   # never read: every call below is refused, or has nothing to do
    good = [p, 0, 2, 3, 100, 300, 100, p, None, 0, 3, p, p, p, p, 1 << 20, None]
    for change, rc in (({"a1": 7}, 1), ({"a3": 0}, 1), ({"a3": 1025}, 2), ({"a4": 0}, 1), ({"a10": 0}, 2), ({"a10": 129}, 2),
                       ({"a4": 1 << 31}, 1), ({"a3": 1024, "a4": 1 << 21}, 1), ({"a2": 1 << 30, "a3": 4}, 1), ({"a2": 40000}, 2),
                       ({"a8": p, "a9": 100}, 1), ({"a8": p, "a9": -1}, 1), ({"a0": None}, 1), ({"a7": None}, 1),
                       ({"a11": None}, 1), ({"a12": None}, 1), ({"a13": None}, 1), ({"a0": odd}, 1), ({"a14": None}, 1),
                       ({"a14": 4104}, 1), ({"a15": 16}, 1), ({"a2": 0}, 0), ({"a2": -1}, 1)):
        assert _call(L.axs6_beam_select, good, **change) == rc, change
        assert rc == 0 or L.axs6_last_error()
    assert L.axs6_beam_select_workspace(0, 3, 100, 3, 0) == 0 and L.axs6_beam_select_workspace(2, 3, 100, 3, 9) == 0
    assert 0 < L.axs6_beam_select_workspace(2, 3, 100, 3, 0) < L.axs6_beam_select_workspace(64, 8, 128000, 16, 1) < 1 << 20


def test_copy_checks_its_arguments():
    L = _lib.lib()
    src, dst = [1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20], [x << 24 for x in range(1, 7)]
    # (2 groups of 3) to (2 of 4), 2 heads of 64
    good = [*src, 0, 2, 3, 4, 2, 64, 5, 4096, 4096, 6, *dst, None]
    for change, rc in (({"a6": 3}, 1), ({"a7": -1}, 1), ({"a8": -1}, 1), ({"a9": -1}, 1), ({"a11": 40}, 2), ({"a11": 272}, 2),
                       ({"a0": None}, 1), ({"a3": None}, 1), ({"a4": None}, 1), ({"a16": None}, 1), ({"a21": None}, 1),
                       ({"a13": None}, 1), ({"a14": None}, 1), ({"a4": src[4] + 8}, 1), ({"a16": dst[0] + 4}, 1),
                       ({"a16": src[0]}, 1), ({"a20": src[4] + 16}, 1), ({"a17": src[0] + 64}, 1),       # shared memory
                       ({"a7": 0}, 0), ({"a9": 0}, 0), ({"a12": 0}, 0), ({"a15": 0}, 0), ({"a10": 0}, 0)):
        assert _call(L.axs6_kv_copy, good, **change) == rc, change
    # in place: the same sequences, at most 4096 a group
    far = [x << 32 for x in range(1, 7)]
    assert L.axs6_kv_copy(*far, 0, 1, 4097, 4097, 1, 16, 1, 4096, 4096, 1, *far, None) == 2
    assert L.axs6_kv_copy(*far, 0, 1, 4, 5, 1, 16, 1, 4096, 4096, 1, *far, None) == 1


def test_shared_attention_checks_its_arguments():
    L = _lib.lib()
    p, st = 4096, _i64(256, 64, 64)
    need = L.axs6_kv_shared_attention_workspace(0, 2, 3, 1, 4, 2, 64, 8, 2)
    assert need > 0
    good = [p, 0, 2, 3, 1, 4, 2, 64, st, p, p, p, p, 8, p, p, p, p, p, 2, p, 0.1, p, p, need, None]
    for change, rc in (({"a1": 3}, 1), ({"a2": -1}, 1), ({"a3": -1}, 1), ({"a5": 3}, 1), ({"a7": 40}, 2), ({"a9": None}, 1),
                       ({"a15": None}, 1), ({"a13": 0}, 1), ({"a14": None}, 1), ({"a20": None}, 1), ({"a21": math.nan}, 1),
                       ({"a22": None}, 1), ({"a23": None}, 1), ({"a23": 4104}, 1), ({"a24": need - 1}, 1), ({"a0": 4097}, 1),
                       ({"a4": 1 << 25, "a24": 1 << 50}, 1), ({"a2": 1 << 20, "a3": 1 << 20}, 1), ({"a4": 0}, 0), ({"a2": 0}, 0)):
        assert _call(L.axs6_kv_shared_attention, good, **change) == rc, change
    assert L.axs6_kv_shared_attention_workspace(0, 0, 3, 1, 4, 2, 64, 8, 2) == 0
    assert L.axs6_kv_shared_attention_workspace(0, 2, 3, 1, 4, 2, 64, 0, 2) == 0
