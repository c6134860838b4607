"""Refusals of the quantised cache's calls that answer before any GPU work: numbers whose sums pass 64 bits, and what
the Python module checks itself (no GPU)."""
from __future__ import annotations

import ctypes

import pytest

from test_kv_abi import abi, batch, cache, calls  # noqa: F401

I64_MAX = (1 << 63) - 1


@pytest.mark.parametrize("window", [I64_MAX, I64_MAX - 1, 1 << 62, (1 << 32) + 1, 121])
@pytest.mark.parametrize("n", [1, 2, 21])
def test_a_ring_refuses_every_window_that_passes_its_cells(abi, window, n):
    ring = cache(abi, ring=1, sinks=8)  # 120 cells go round
    nothing = batch(abi, n_seqs=0, n_tokens=0, starts=4096, max_len=n)
    assert calls(abi, ring, nothing, window=window, which="a") == [abi.ERR_INVALID_ARG]
    assert "ring" in abi.last_error()[1]
    assert calls(abi, cache(abi), nothing, window=window, which="a") == [abi.OK]  # a plain cache: its whole prefix


@pytest.mark.parametrize("window", [I64_MAX, 1 << 62, (1 << 32) + 1, 120])
def test_a_chain_refuses_every_window_that_passes_its_ring(abi, window):
    p = 4096  # never read: the call answers first
    layers = (abi.Layer * 1)(abi.Layer(*[p] * 9))
    norms = (ctypes.c_void_p * 1)(p)
    norms = ctypes.cast(norms, ctypes.POINTER(ctypes.c_void_p))
    attention = abi.AttentionDesc(1e4, 128, 1, norms, norms)
    desc = abi.ChainDesc(1, 256, 4, 2, 64, 512, 1e-6, 2, 0, ctypes.cast(layers, ctypes.POINTER(abi.Layer)), p, 64,
                         ctypes.pointer(attention), None)
    kvd = abi.ChainKVDesc(abi.KV_Q8_0, abi.KV_Q8_0, window, 8, 1)
    handle = ctypes.c_void_p()
    got = abi.lib().b200q8_chain_create_kv(ctypes.byref(desc), ctypes.byref(kvd), 0, ctypes.byref(handle))
    assert got == abi.ERR_INVALID_ARG and "ring" in abi.last_error()[1]
