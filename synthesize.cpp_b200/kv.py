"""A quantised key/value cache and the attention that reads it, over the C ABI.

* ``write(cache, k, v, pos, ...)``   rows of keys and values enter the cache as Q4_0 or Q8_0 blocks
* ``read(cache, n, pos, ...)``       the same rows back as floating-point rows
* ``attend(cache, q, pos, ...)``     attention over the cached prefix, whole or as a sliding window plus the
                                     first ``cache.sinks`` positions

The cache's four arrays belong to the caller (``new_cache`` allocates them with torch); their layout is the one
include/b200q8.h documents at b200q8_kv_cache.  Every call names its rows by runs of consecutive positions: run i is
rows ``starts[i]:starts[i+1]`` at positions ``pos[i]``, ``pos[i] + 1``, ... of slot ``slots[i]``; without ``starts``
each run is one row, without ``slots`` run i is slot i; ``max_len`` bounds the runs' lengths (left out, the number of rows does; a close bound
makes a faster call).  ``pos``, ``slots`` and ``starts`` are int32 CUDA tensors.  Work is enqueued on torch's current
stream of the cache's device, whichever device is current; a failure raises B200Q8Error, and what only the device can see
(a position outside the cache) is reported by ``q8.device_status``.  Rows that no run names are left alone: where a call
allocates its result, they hold whatever the memory held.  Nothing here is recorded for gradients.
"""
from __future__ import annotations

import torch

from ._abi import KV_Q4_0, KV_Q8_0, KVBatch, KVCacheDesc, B200Q8Error, check, lib
from .q8 import SRC_TYPES

__all__ = ["KV_Q4_0", "KV_Q8_0", "KVCache", "B200Q8Error", "new_cache", "write", "read", "attend"]

_TYPE_OF = {torch.uint8: KV_Q4_0, torch.int8: KV_Q8_0}
_BLOCK_BYTES = {torch.uint8: 16, torch.int8: 32}


class KVCache:
    """Four CUDA tensors: codes [n_slots, n_kv, n_ctx, row] (uint8 rows of head_dim / 2 bytes are Q4_0, int8 rows of
    head_dim bytes are Q8_0) and float16 scales [n_slots, n_kv, n_ctx, head_dim / 32], for keys and for values."""

    __slots__ = ("k_codes", "k_scales", "v_codes", "v_scales", "n_kv", "head_dim", "_device", "_desc")

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                 sinks: int = 0, ring: bool = False):
        n_slots, n_kv, n_ctx, nb = shape = k_scales.shape
        dev = k_codes.get_device()
        for codes, scales in ((k_codes, k_scales), (v_codes, v_scales)):
            if (dev < 0 or codes.dtype not in _BLOCK_BYTES or scales.dtype != torch.float16 or scales.shape != shape
                    or codes.shape != (n_slots, n_kv, n_ctx, _BLOCK_BYTES[codes.dtype] * nb)
                    or codes.get_device() != dev or scales.get_device() != dev
                    or not codes.is_contiguous() or not scales.is_contiguous()):
                raise ValueError("KVCache: codes must be contiguous uint8 [n_slots, n_kv, n_ctx, head_dim/2] or int8 "
                                 "[..., head_dim] CUDA tensors and scales float16 [n_slots, n_kv, n_ctx, head_dim/32]")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.n_kv, self.head_dim, self._device = n_kv, 32 * nb, dev
        self._desc = KVCacheDesc(_TYPE_OF[k_codes.dtype], _TYPE_OF[v_codes.dtype], n_slots, n_ctx, n_kv, 32 * nb, sinks,
                                 1 if ring else 0, k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
                                 v_scales.data_ptr())

    @property
    def n_slots(self) -> int:
        return self._desc.n_slots

    @property
    def n_ctx(self) -> int:
        return self._desc.n_ctx

    @property
    def sinks(self) -> int:
        return self._desc.sinks

    @property
    def ring(self) -> bool:
        return self._desc.ring != 0


def new_cache(n_slots: int, n_ctx: int, n_kv: int, head_dim: int, type_k: int = KV_Q8_0, type_v: int = KV_Q8_0,
              sinks: int = 0, ring: bool = False, device: torch.device | str = "cuda") -> KVCache:
    """Allocates a cache (n_ctx is rounded up to a multiple of 64)."""
    if head_dim % 32 != 0 or not 32 <= head_dim <= 256:
        raise ValueError("new_cache: head_dim must be a multiple of 32 up to 256")
    n_ctx = (n_ctx + 63) // 64 * 64
    arrays = []
    for t in (type_k, type_v):
        if t not in (KV_Q4_0, KV_Q8_0):
            raise ValueError("new_cache: types are KV_Q4_0 or KV_Q8_0")
        row, dt = (head_dim // 2, torch.uint8) if t == KV_Q4_0 else (head_dim, torch.int8)
        arrays.append(torch.zeros((n_slots, n_kv, n_ctx, row), dtype=dt, device=device))
        arrays.append(torch.zeros((n_slots, n_kv, n_ctx, head_dim // 32), dtype=torch.float16, device=device))
    return KVCache(*arrays, sinks=sinks, ring=ring)


def _batch(cache: KVCache, n_tokens: int, pos, slots, starts, max_len: int | None, window: int = 1) -> KVBatch:
    dev, i32 = cache._device, torch.int32
    n = pos.numel()
    # dense vectors of int32 on the cache's device
    if (pos.dtype != i32 or pos.get_device() != dev or pos.dim() != 1 or not pos.is_contiguous()
            or slots is not None and (slots.dtype != i32 or slots.get_device() != dev or slots.shape != pos.shape
                                      or not slots.is_contiguous())
            or starts is not None and (starts.dtype != i32 or starts.get_device() != dev or starts.dim() != 1
                                       or starts.numel() != n + 1 or not starts.is_contiguous())):
        raise ValueError("kv: pos, slots [n] and starts [n + 1] must be dense int32 tensors on the cache's device")
    if starts is None:
        return KVBatch(n, n_tokens, 1, None, pos.data_ptr(), None if slots is None else slots.data_ptr())
    if max_len is None:  # no run is longer than all rows, and in a ring than its cells allow
        most = cache.n_ctx - cache.sinks - window + 1 if cache.ring else n_tokens
        max_len = max(1, min(n_tokens, most))
    return KVBatch(n, n_tokens, max_len, starts.data_ptr(), pos.data_ptr(),
                   None if slots is None else slots.data_ptr())


def _rows(cache: KVCache, t: torch.Tensor, heads: int, what: str) -> int:
    """Checks rows [n, heads, head_dim] (or [n, heads * head_dim]); returns their stride in bytes."""
    hd, shape, stride = cache.head_dim, t.shape, t.stride()
    if len(shape) == 3:
        dense = shape[1] == heads and shape[2] == hd and stride[2] == 1 and (heads == 1 or stride[1] == hd)
    else:
        dense = len(shape) == 2 and shape[1] == heads * hd and stride[1] == 1
    if not dense or t.dtype not in SRC_TYPES or t.get_device() != cache._device:
        raise ValueError(f"kv: {what} must be float32, float16 or bfloat16 [n, {heads}, {hd}] with dense rows, on the "
                         "cache's device")
    return stride[0] * t.element_size()


def write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor | None = None,
          starts: torch.Tensor | None = None, max_len: int | None = None) -> None:
    """Quantises rows k, v [n, n_kv, head_dim] (row-strided views allowed) into their cells."""
    dev = cache._device
    if torch._C._cuda_getDevice() != dev:  # the library launches on the current device
        with torch.cuda.device(dev):
            return write(cache, k, v, pos, slots, starts, max_len)
    n = k.shape[0]
    if k.dtype != v.dtype or n != v.shape[0]:
        raise ValueError("kv.write: k and v must have one type and as many rows")
    ks, vs = _rows(cache, k, cache.n_kv, "k"), _rows(cache, v, cache.n_kv, "v")
    check(lib().b200q8_kv_write(cache._desc, _batch(cache, n, pos, slots, starts, max_len), k.data_ptr(), ks,
                                v.data_ptr(), vs, SRC_TYPES[k.dtype], torch._C._cuda_getCurrentRawStream(dev)))


def read(cache: KVCache, n: int, pos: torch.Tensor, slots: torch.Tensor | None = None,
         starts: torch.Tensor | None = None, max_len: int | None = None, dtype: torch.dtype = torch.float32,
         out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The n rows of the runs as values: (k, v), each [n, n_kv, head_dim]."""
    dev = cache._device
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return read(cache, n, pos, slots, starts, max_len, dtype, out)
    if out is None:
        both = cache.k_scales.new_empty((2, n, cache.n_kv, cache.head_dim), dtype=dtype)
        k, v = out = both.unbind(0)
        ks = vs = cache.n_kv * cache.head_dim * both.element_size()
    else:
        k, v = out
        if k.dtype != v.dtype or k.shape[0] != n or v.shape[0] != n:
            raise ValueError("kv.read: out must be two tensors of n rows of one type")
        ks, vs = _rows(cache, k, cache.n_kv, "out"), _rows(cache, v, cache.n_kv, "out")
    if k.dtype not in SRC_TYPES:
        raise ValueError("kv.read: dtype must be float32, float16 or bfloat16")
    check(lib().b200q8_kv_read(cache._desc, _batch(cache, n, pos, slots, starts, max_len), k.data_ptr(), ks,
                               v.data_ptr(), vs, SRC_TYPES[k.dtype], torch._C._cuda_getCurrentRawStream(dev)))
    return out


def attend(cache: KVCache, q: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor | None = None,
           starts: torch.Tensor | None = None, max_len: int | None = None, window: int = 0, scale: float = 0.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [n, n_head, head_dim] over the cached positions each row sees; returns [n, n_head, head_dim] in
    q's type.  window 0 sees the whole prefix; scale 0 means 1/sqrt(head_dim)."""
    dev = cache._device
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return attend(cache, q, pos, slots, starts, max_len, window, scale, out)
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("kv.attend: q must be [n, n_head, head_dim]")
    n, heads, _ = shape
    qs = _rows(cache, q, heads, "q")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os_ = heads * cache.head_dim * q.element_size()
    elif out.dtype != q.dtype or out.shape[0] != n:
        raise ValueError("kv.attend: out must have q's rows and type")
    else:
        os_ = _rows(cache, out, heads, "out")
    check(lib().b200q8_kv_attend(cache._desc, _batch(cache, n, pos, slots, starts, max_len, window), q.data_ptr(), qs,
                                 out.data_ptr(), os_, SRC_TYPES[q.dtype], heads, window, scale, torch._C._cuda_getCurrentRawStream(dev)))
    return out
