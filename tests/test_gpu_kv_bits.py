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


# --------------------------------------------------------------------------- scores and value scales set one by one


def scored(kv, dev, n_kv, hd, n_ctx, scores, bits_k=8, bits_v=8, seed=5):
    """(cache, first): one slot, whose cell j scores scores[j] (to fp16) with a query whose value 0 is first and with
    any other values: keys hold a one there and zeros elsewhere."""
    c = make(kv, dev, 1, n_ctx, n_kv, hd, bits_k, bits_v, seed=seed)
    s = torch.as_tensor(scores, dtype=torch.float64, device=dev)
    zero, one = (0x88, 1) if bits_k == 4 else (0, 1)
    c.k_codes[:] = zero
    c.k_codes[0, :, :len(s), 0] = torch.where(s < 0, zero - one, zero + one).to(c.k_codes.dtype)
    c.k_scales[0, :, :len(s)] = s.abs()[None, :, None].half()
    assert R.places(hd, 4)[0] == 0
    return c, hd ** 0.5


def single(kv, c, first, nh, p, dtype=F32, window=0):
    """The row at position p, over the kernels' and the plain form's results: (got, want, mass, reach)."""
    dev = c.k_codes.device
    q = rows(dev, 1, nh, c.head_dim, dtype, seed=77)
    q[:, :, 0] = first
    got = kv.attend(c, q, i32(dev, p), window=window)
    return (got, *R.attend(c, q, [p], [0], [1], window))


# query heads, kv heads, head size, cells, position: four warps a CTA, eight (long caches of few heads), the same for
# a size of three blocks, one of two, one of one; several steps a warp; then the general kernel's forms for single rows
SINGLES = [(16, 8, 128, 512, 300), (4, 2, 128, 8192, 6100), (4, 2, 96, 8192, 6100), (4, 2, 64, 8192, 6100),
           (16, 8, 64, 512, 300), (4, 4, 32, 512, 300), (128, 64, 128, 2048, 2000), (16, 2, 128, 512, 300),
           (4, 2, 256, 512, 300)]


@pytest.mark.parametrize("bits_k,bits_v", [(4, 4), (8, 8), (8, 4), (4, 8)])
@pytest.mark.parametrize("nh,n_kv,hd,n_ctx,p", SINGLES)
@pytest.mark.parametrize("above", [45.0, 80.0, 150.0])
def test_a_zero_valued_cell_of_high_score(kv, dev, nh, n_kv, hd, n_ctx, p, bits_k, bits_v, above):
    """A cell whose values are all zero (a sink) takes nearly all the weight, wherever it lies among the cells that
    warps and CTAs share out, first values of zero or not: results are what the others' share leaves."""
    g = torch.Generator().manual_seed(nh + hd)
    for zeros in ([0], [45], [p], [p // 2], [p // 2, p // 2 + 33, p - 70], list(range(40)) + [p - 9]):
        s = torch.randn(p + 1, generator=g)
        s[zeros[-1]] = above
        c, first = scored(kv, dev, n_kv, hd, n_ctx, s, bits_k, bits_v)
        c.v_scales[0, :, zeros] = 0.0
        got, want, mass, reach = single(kv, c, first, nh, p)
        # weights times value scales of below 2^-32 of the largest weight and scale lose bits; a cell brings 127 at most
        most = R.values_of(c.v_codes[0, :, :p + 1], c.v_scales[0, :, :p + 1], "v").abs().amax()
        tol = R.tolerance(want, mass, reach, F32) + (p + 1) * 2.0 ** -32 * most
        assert torch.isfinite(got).all(), zeros
        assert ((got.double() - want).abs() <= tol).all(), zeros


@pytest.mark.parametrize("nh,n_kv,hd,n_ctx,p", SINGLES[:7])
def test_single_rows_hold_products_of_weight_and_value_scale(kv, dev, nh, n_kv, hd, n_ctx, p):
    """Large value scales at negligible weights, or large weights at values of zero, cost the products that count no
    bits, in one step of the kernel or in steps one after another."""
    tiny = 177 * 2.0 ** -24  # with few bits to spare in fp16
    for at in ([3], [40], [p - 3], [3, 40, p - 40]):
        s = torch.zeros(p + 1)
        s[at] = -40.0
        c, first = scored(kv, dev, n_kv, hd, n_ctx, s)
        c.v_scales[0] = tiny
        c.v_scales[0, :, at] = 32768.0
        got, want, mass, reach = single(kv, c, first, nh, p)
        assert ((got.double() - want).abs() <= R.tolerance(want, mass, reach, F32)).all(), at
        s[at] = 45.0  # 65 octaves above
        c, first = scored(kv, dev, n_kv, hd, n_ctx, s)
        c.v_scales[0, :, at] = 0.0
        got, want, mass, reach = single(kv, c, first, nh, p)
        assert ((got.double() - want).abs() <= R.tolerance(want, mass, reach, F32)).all(), at


@pytest.mark.parametrize("t,nh,n_kv,hd,n_ctx,p", [(1, 1024, 256, 128, 512, 300), (1, 512, 256, 256, 512, 300),
                                                  (9, 512, 256, 64, 512, 300), (9, 512, 256, 128, 512, 300),
                                                  (1, 768, 256, 160, 512, 300)])
def test_early_large_value_scales_cost_later_steps_nothing(kv, dev, t, nh, n_kv, hd, n_ctx, p):
    """... in the general kernel: a warp's first step holds value scales 2^30 above the others', at negligible weights
    (so many heads that cells are not split)."""
    s = torch.zeros(p + t)
    s[:128] = -60.0
    c, first = scored(kv, dev, n_kv, hd, n_ctx, s)
    c.v_scales[0] = 177 * 2.0 ** -24
    c.v_scales[0, :, :128] = 32768.0
    q = rows(dev, t, nh, hd, seed=78)
    q[:, :, 0] = first
    got = kv.attend(c, q, i32(dev, p), None, i32(dev, 0, t), t)
    want, mass, reach = R.attend(c, q, [p], [0], [t], 0)
    assert ((got.double() - want).abs() <= R.tolerance(want, mass, reach, F32)).all()


@pytest.mark.parametrize("bits_v", [4, 8])
@pytest.mark.parametrize("nh,n_kv,hd", [(64, 32, 128), (64, 32, 64)])
def test_prompts_after_early_large_value_scales(kv, dev, nh, n_kv, hd, bits_v):
    """... and in the 128-row kernel, up and down more than once along the prefix."""
    p, t = 500, 130
    s = torch.zeros(p + t)
    for first in (0, 192, 384):
        s[first:first + 64] = -60.0
    c, first = scored(kv, dev, n_kv, hd, 640, s, 8, bits_v)
    c.v_scales[0] = 177 * 2.0 ** -24
    c.v_scales[0, :, 0:64] = 32768.0
    c.v_scales[0, :, 192:256] = 8.0
    c.v_scales[0, :, 384:448] = 1000.0
    q = rows(dev, t, nh, hd, seed=79)
    q[:, :, 0] = first
    got = kv.attend(c, q, i32(dev, p), None, i32(dev, 0, t), t)
    want, mass, reach = R.attend(c, q, [p], [0], [t], 0)
    assert ((got.double() - want).abs() <= R.tolerance(want, mass, reach, F32)).all()


@pytest.mark.parametrize("t,nh,n_kv,hd", [(1, 16, 8, 128), (1, 4, 2, 96), (1, 16, 2, 128), (9, 4, 2, 128), (3, 4, 2, 256),
                                          (130, 64, 32, 128)])
def test_an_infinite_key_scale_spoils_who_sees_it(kv, dev, t, nh, n_kv, hd):
    """Codes of both signs times infinity: the score is not a number, whatever the codes' own sum."""
    c = make(kv, dev, 1, 320, n_kv, hd, 8, 8, seed=80)
    q = rows(dev, t, nh, hd, seed=81)
    for p, hurt in ((100, t > 60), (160, True)):
        c.k_scales[0, :, 160, 0] = float("inf")
        got = kv.attend(c, q, i32(dev, p), None, i32(dev, 0, t), t)
        bad = torch.arange(p, p + t, device=dev) >= 160
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all() and bool(bad.any()) == hurt


@pytest.mark.parametrize("bits_k", [4, 8])
@pytest.mark.parametrize("nh,n_kv,hd,n_ctx,p", SINGLES)
def test_a_strong_query_channel_that_keys_do_not_meet(kv, dev, nh, n_kv, hd, n_ctx, p, bits_k):
    """A value of q 2^12 times the others where keys are zero: the others keep their bits."""
    c = make(kv, dev, 1, n_ctx, n_kv, hd, bits_k, 8, seed=90)
    at = R.places(hd, 4)[7]
    if bits_k == 8:
        c.k_codes[..., at] = 0
    else:
        byte = c.k_codes[..., at // 2]
        c.k_codes[..., at // 2] = byte & (0x0f if at % 2 else 0xf0) | (0x80 if at % 2 else 0x08)
    c.k_scales[:] *= 4.0
    q = rows(dev, 1, nh, hd, seed=91)
    q[:, :, 7] = 4096.0
    got = kv.attend(c, q, i32(dev, p))
    want, mass, reach = R.attend(c, q, [p], [0], [1], 0)
    err, tol = (got.double() - want).abs(), R.tolerance(want, mass, reach, F32)
    assert (err <= tol).all(), float((err / tol).max())
