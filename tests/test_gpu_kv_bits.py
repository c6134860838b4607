"""How exact b200q8_kv_attend is where scores, value scales and types leave the ordinary: against the plain 64-bit form."""
from __future__ import annotations

import pytest
import torch

import kv_reference as R
from test_gpu_kv import BF16, F32, TYPES, i32, kv, make, no_device_error, rows, starts_of  # noqa: F401

pytestmark = pytest.mark.gpu


def rounded(got, want, mass, reach):
    """got is a result as exact as F32 rows' are, rounded once: rounding keeps order, so it lies between the bound's
    two ends rounded."""
    bound = R.tolerance(want, mass, reach, F32)
    lo, hi = ((want + s * bound).to(got.dtype) for s in (-1, 1))
    return (lo <= got) & (got <= hi)


@pytest.mark.parametrize("bits_k,bits_v", [(4, 4), (8, 8), (8, 4), (4, 8)])
@pytest.mark.parametrize("nh,n_kv,hd,n_ctx,lens,pos", [
    (32, 16, 128, 320, [130, 64, 7], [60, 200, 300]),  # the 128-row kernel
    (80, 16, 64, 320, [90, 64, 7], [60, 200, 300]),
    (8, 2, 128, 320, [33, 5, 18], [60, 200, 300]),     # 16 rows a warp
    (6, 2, 64, 320, [33, 5, 18], [60, 200, 300]),
    (16, 8, 128, 320, [1, 1, 1], [60, 200, 300]),      # single rows
])
def test_bf16_rows_are_f32_results_rounded_once(kv, dev, bits_k, bits_v, nh, n_kv, hd, n_ctx, lens, pos):
    c = make(kv, dev, 3, n_ctx, n_kv, hd, bits_k, bits_v, seed=hd + nh)
    q = rows(dev, sum(lens), nh, hd, BF16, seed=nh + 1)
    got = kv.attend(c, q, i32(dev, *pos), i32(dev, 2, 0, 1), starts_of(dev, lens), max(lens))
    want, mass, reach = R.attend(c, q, pos, [2, 0, 1], lens, 0)
    ok = rounded(got, want, mass, reach)
    assert ok.all(), float((~ok).double().mean())
