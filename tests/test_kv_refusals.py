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


# ------------------------------------------------------------------------------------------------ the Python module


class OnDevice:
    """A CPU tensor that says it is on device 1: enough for the module's checks."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 1

    def __getattr__(self, name):
        return getattr(self.t, name)


class Calls:
    """The library's calls, recording the device that is current when they are made."""

    def __init__(self, state):
        self.state, self.seen, self.batches = state, [], []

    def __getattr__(self, name):
        def call(*args):
            self.seen.append((name, self.state["device"]))
            self.batches.append(args[1])
            return 0

        return call


@pytest.fixture()
def two_devices(pkg, monkeypatch):
    """(kv, a cache on device 1, the calls' record, the state whose "device" is current)."""
    import torch
    from synthesize_cpp_b200 import _abi, kv

    state = {"device": 0}

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index

        def __exit__(self, *_):
            state["device"] = self.before

    lib = Calls(state)
    monkeypatch.setattr(kv, "lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["device"])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index)
    c = object.__new__(kv.KVCache)
    c.n_kv, c.head_dim, c._device = 2, 64, 1
    c._desc = _abi.KVCacheDesc(8, 8, 16, 128, 2, 64, 4, 0, 4096, 4096, 4096, 4096)
    return kv, c, lib, state


@pytest.mark.parametrize("current", [0, 1])
def test_calls_run_on_the_caches_device(two_devices, current):
    import torch

    kv, c, lib, state = two_devices
    state["device"] = current
    x, p = OnDevice(torch.zeros((1, 2, 64))), OnDevice(torch.zeros(1, dtype=torch.int32))
    kv.write(c, x, x, p)
    kv.read(c, 1, p, out=(x, x))
    kv.attend(c, x, p, out=x)
    assert lib.seen == [("b200q8_kv_write", 1), ("b200q8_kv_read", 1), ("b200q8_kv_attend", 1)]
    assert state["device"] == current


def test_runs_without_max_len_are_bounded_by_the_rows(two_devices):
    """A caller who names runs and no bound gets every row, not zeros beyond the first of each run."""
    import torch

    kv, c, lib, _ = two_devices
    ints = lambda *v: OnDevice(torch.tensor(v, dtype=torch.int32))  # noqa: E731
    x, p, starts = OnDevice(torch.zeros((5, 2, 64))), ints(0, 9), ints(0, 3, 5)
    kv.write(c, x, x, p, None, starts)
    kv.read(c, 5, p, None, starts, out=(x, x))
    kv.attend(c, x, p, starts=starts, out=x)
    assert [b.max_len for b in lib.batches] == [5, 5, 5]
    kv.attend(c, x, p, None, starts, 3, out=x)
    kv.attend(c, OnDevice(torch.zeros((2, 2, 64))), p, out=OnDevice(torch.zeros((2, 2, 64))))
    assert [b.max_len for b in lib.batches[3:]] == [3, 1]
    none = OnDevice(torch.zeros((0, 2, 64)))
    kv.attend(c, none, p, None, ints(0, 0, 0), out=none)
    assert lib.batches[-1].max_len == 1
    c._desc.ring = 1  # 124 cells go round
    x = OnDevice(torch.zeros((200, 2, 64)))
    kv.write(c, x, x, p, None, starts)
    kv.attend(c, x, p, None, starts, window=100, out=x)
    kv.attend(c, x, p, None, starts, window=124, out=x)
    assert [b.max_len for b in lib.batches[-3:]] == [124, 25, 1]


@pytest.mark.parametrize("head_dim", [33, 63, 0, 16, 48, 288, -32])
def test_new_cache_refuses_other_head_sizes(pkg, head_dim):
    """... 33 in four bits is 16 bytes a row, as 32 is."""
    from synthesize_cpp_b200 import kv

    for t in (kv.KV_Q4_0, kv.KV_Q8_0):
        with pytest.raises(ValueError, match="multiple of 32"):
            kv.new_cache(1, 64, 1, head_dim, t, t, device="cpu")
