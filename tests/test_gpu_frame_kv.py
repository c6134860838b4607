"""Steps with output heads, frames and long caches over quantised caches: what b200q8_chain_create_kv's chains share
with the others."""
from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from test_gpu_attention import THETA, qk_norms
from test_gpu_chain import EPS, H, HD, I, NH, NKV, make_model, upload
from test_gpu_chain_kv import build, check_layer, i32
from test_gpu_frame import G, PV, TV, rms_norm, t

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv(pkg):
    return importlib.import_module("synthesize_cpp_b200.kv")


def stack(O, chain_mod, dev, seed, vocab, n_heads, table_rows, n_slots, max_m, kvd):
    mats, norms, _ = make_model(O, 2, seed=seed)
    qkn = qk_norms(O, 2, seed + 50)
    table = O.quantize_rows(O.normal(seed + 70, table_rows * H, 0.5).reshape(table_rows, H))
    out_norm = (1.0 + 0.1 * O.normal(seed + 71, H)).astype(np.float32)
    heads = [O.quantize_rows(O.normal(seed + 80 + i, vocab * H, 0.02).reshape(vocab, H)) for i in range(n_heads)]
    layers, t_table = upload(mats, norms, table, dev)
    for l, L in enumerate(layers):
        L["q_norm"], L["k_norm"] = t(qkn[2 * l], dev), t(qkn[2 * l + 1], dev)
    ch = chain_mod.DecodeChain(layers, t_table, hidden=H, n_head=NH, n_kv=NKV, head_dim=HD, inter=I, eps=EPS,
                               max_m=max_m, attention=dict(rope_theta=THETA, n_ctx=64, n_slots=n_slots, kv=kvd),
                               output=dict(norm=t(out_norm, dev), heads=[t(h, dev) for h in heads]))
    return ch, dict(table=table, out_norm=out_norm, heads=heads)


@pytest.mark.parametrize("m", [1, 3, 12])
def test_step_output_stage(chain_mod, O, dev, m):
    """The heads' logits from the step's own hidden rows, as for F32 caches; run_at gives the same residual stream."""
    ch, ref = stack(O, chain_mod, dev, 3000, 512, 2, 64, m, 16, dict(type_k=8, type_v=2))
    other, _ = stack(O, chain_mod, dev, 3000, 512, 2, 64, m, 16, dict(type_k=8, type_v=2))
    rng = np.random.default_rng(m)
    h, hid, lg = (torch.empty((m, n), device=dev) for n in (H, H, 512))
    plain = torch.empty((m, H), device=dev)
    for step in range(3):
        x, ids = t(rng.standard_normal((m, H)).astype(np.float32), dev), t(rng.integers(0, 64, m).astype(np.int32), dev)
        pos = i32(dev, [step] * m)
        ch.step(ids=ids, x_in=x, pos=pos, h_out=h, hidden_out=hid, logits=lg, head=step % 2)
        other.run_at(ids, x, pos, plain)
        torch.cuda.synchronize(dev)
        assert torch.equal(h, plain)
        hidg = hid.cpu().numpy()
        assert np.array_equal(hidg, rms_norm(h.cpu().numpy(), ref["out_norm"]))
        y, bound = O.mul_mat(ref["heads"][step % 2], H, hidg)
        assert np.all(np.abs(lg.cpu().numpy().astype(np.float64) - y) <= 1e-5 * bound + 1e-30)
    ch.close()
    other.close()


@pytest.mark.parametrize("m", [1, 3])
def test_frames(chain_mod, frame_mod, O, q8, dev, m):
    """Frames (the predictor's prefill gives a slot two rows in one step) equal the same steps made one by one, bit
    for bit; the talker's ring goes past its cells."""
    ring = dict(type_k=8, type_v=8, window=40, sinks=2, ring=True)
    plain = dict(type_k=8, type_v=2)
    talker, tref = stack(O, chain_mod, dev, 4000, TV, 1, TV, m, 8, ring)
    pred, _ = stack(O, chain_mod, dev, 5000, PV, G - 1, 8, m, 8, plain)
    talker2, _ = stack(O, chain_mod, dev, 4000, TV, 1, TV, m, 8, ring)
    pred2, _ = stack(O, chain_mod, dev, 5000, PV, G - 1, 8, m, 8, plain)
    ptables = [O.quantize_rows(O.normal(6000 + g, PV * H, 0.5).reshape(PV, H)) for g in range(G - 1)]
    tables = [t(p, dev) for p in ptables]
    fr = frame_mod.Frame(talker, pred, tables)
    rng = np.random.default_rng(11 + m)
    slots = np.arange(m, dtype=np.int32)[::-1].copy()
    prev = np.stack([rng.integers(0, TV, m)] + [rng.integers(0, PV, m) for _ in range(G - 1)], 1).astype(np.int32)
    codes = torch.empty((m, G), dtype=torch.int32, device=dev)
    hid, tlog = torch.empty((m, H), device=dev), torch.empty((m, TV), device=dev)
    hid2, tlog2, plog = torch.empty_like(hid), torch.empty_like(tlog), torch.empty((2 * m, PV), device=dev)
    for f in range(72):
        text = rng.standard_normal((m, H)).astype(np.float32)
        pos = t(np.full(m, f, np.int32), dev)
        fr.run(codes, text=t(text, dev), prev=t(prev, dev), pos=pos, slots=t(slots, dev), hidden=hid, talker_logits=tlog)
        got = codes.cpu().numpy()
        x = O.get_rows(ptables[0], H, prev[:, 1])[0].astype(np.float32)
        for g in range(2, G):
            x = x + O.get_rows(ptables[g - 1], H, prev[:, g])[0]
        x = (x + O.get_rows(tref["table"], H, prev[:, 0])[0]) + text
        talker2.step(x_in=t(x, dev), pos=pos, slots=t(slots, dev), hidden_out=hid2, logits=tlog2)
        assert torch.equal(hid, hid2) and torch.equal(tlog, tlog2), f
        cur = tlog2.argmax(-1).int()
        assert np.array_equal(got[:, 0], cur.cpu().numpy()), f
        both = np.empty((2 * m, H), np.float32)
        both[0::2], both[1::2] = hid2.cpu().numpy(), O.get_rows(tref["table"], H, got[:, 0].astype(np.int32))[0]
        pred2.step(x_in=t(both, dev), pos=i32(dev, [0, 1] * m), slots=t(np.repeat(slots, 2), dev), logits=plog)
        for g in range(1, G):
            lg = plog[1::2] if g == 1 else plog[:m]
            assert np.array_equal(got[:, g], lg.argmax(-1).int().cpu().numpy()), (f, g)
            if g + 1 < G:
                pred2.step(ids=t(got[:, g], dev), table=tables[g - 1], pos=i32(dev, [g + 1] * m),
                           slots=t(slots, dev), logits=plog[:m], head=g)
        prev = got
    assert q8.device_status(0, clear=True) == 0
    fr.close()
    for ch in (talker, pred, talker2, pred2):
        ch.close()


def test_long_caches_at_every_batch_size(pkg, O, kv, chain_mod, q8, dev):
    """4096 cells a slot: steps of one token and of more take kernels of their own, each first met in a capture (the
    positions stay where check_layer's bound on the rotation holds)."""
    ch, qkn = build(O, chain_mod, dev, 1, 12, 4096, 6, 2600, dict(type_k=8, type_v=8))
    c = ch.kv_cache(0)
    k = torch.randn((60, NKV, HD), device=dev)
    for s in range(6):
        kv.write(c, k.roll(s, 0), k.roll(-s, 0), i32(dev, [0]), i32(dev, [s]), i32(dev, [0, 60]), 60)
    rng = np.random.default_rng(9)
    for step, m in enumerate((2, 1, 5, 3, 4, 6)):
        pos, slots = [60 - 7 * i + step for i in range(m)], [(5 * i + step) % 6 for i in range(m)]
        x = torch.from_numpy(rng.standard_normal((m, H)).astype(np.float32)).to(dev)
        h = torch.empty((m, H), device=dev)
        ch.run_at(i32(dev, rng.integers(0, 64, m)), x, i32(dev, pos), h, slots=i32(dev, slots))
        torch.cuda.synchronize(dev)
        check_layer(O, kv, ch, qkn, 0, m, pos, slots, 0, dev)
    assert q8.device_status(0, clear=True) == 0
    ch.close()
