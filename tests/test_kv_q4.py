"""The paged 4-bit cache on the CPU: its definition (the oracle against plain formulas and
planted mistakes), and the refusals of its entry points, which come before any device work."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import kv_q4_oracle as orc
import questwend_amd as qa

OK, INVALID, UNSUPPORTED, NOT_READY = 0, -1, -2, -5


def test_quantizer_is_nearest_and_keeps_the_largest():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)).astype(np.float32) * np.exp(rng.uniform(-6, 6, (50, 1))).astype(np.float32)
    code, d = orc.quantize(x)
    assert code.min() == 0 and code.max() <= 15
    v = orc.values(code, d)
    dd = np.repeat(np.abs(orc.as_f64(d)), 32, axis=1)
    # nearest, but for what the clamp at 7 cuts off on the other side of the largest value
    assert np.all(np.abs(v - x) <= np.where(np.abs(x) >= 7.5 * dd, 1.01 * dd, 0.5 * dd * (1 + 1e-9)))
    # the largest value of a block is kept to the scale's rounding (2^-11)
    y, w = x.reshape(50, 4, 32), v.reshape(50, 4, 32)
    at = np.abs(y).argmax(-1)[..., None]
    a, b = np.take_along_axis(y, at, -1), np.take_along_axis(w, at, -1)
    assert np.all(np.abs(a - b) <= np.abs(a) * 2.0**-11)


def test_quantizer_edges():
    x = np.zeros((6, 32), np.float32)
    x[1, 3] = np.inf
    x[2, 5] = np.nan
    x[3, :2] = [4.0, -4.0]          # a tie: the positive one
    x[4, 0] = 3e38                  # beyond f16's scales
    x[5, 0] = 1e-9                  # below them
    code, d = orc.quantize(x)
    v = orc.values(code, d)
    assert np.all(v[0] == 0) and np.all(np.isnan(v[1])) and np.all(np.isnan(v[2]))
    assert v[3, 0] == 4.0 and v[3, 1] == -3.5
    assert v[4, 0] == 8 * 65504.0 and np.all(v[5] == 0)


@pytest.mark.parametrize("D,P", [(64, 32), (128, 64), (256, 128)])
def test_layout_places_are_distinct_and_round_trip(D, P):
    c = orc.Cache(2, 2, D, P)
    for tab in c.tables():
        seen = set()
        for place, scales in tab:
            seen |= {(int(a), int(s)) for a, s in place}
            seen |= {(int(a), -1) for a in scales}
        assert len(seen) == 32 * (D + D // 32)
        assert max(a for a, _ in seen) < 36 * D
    rng = np.random.default_rng(1)
    slots = rng.permutation(2 * P)[:40]
    k, v = rng.standard_normal((2, 40, 2, D)).astype(np.float32)
    c.store(k, v, slots)
    for x, y in zip((k, v), c.load(slots)):
        assert np.array_equal(y, orc.values(*orc.quantize(x)))
    before = c.load(slots[3:4])[0].copy()
    place, _ = c.tables()[0][int(slots[3]) % P % 32]
    c.data[c.cell(int(slots[3]), 1) + place[7, 0]] ^= 1 << int(place[7, 1])   # a planted mistake
    assert not np.array_equal(before, c.load(slots[3:4])[0])


def test_attention_of_equal_keys_is_the_mean():
    rng = np.random.default_rng(2)
    k, v = np.ones((9, 1, 64)), rng.standard_normal((9, 1, 64))
    q = rng.standard_normal((2, 3, 64))
    out, _, _ = orc.attention(q, k, v, 2, 0.125)
    assert np.allclose(out[1], v[:, 0].mean(0)) and np.allclose(out[0], v[:8, 0].mean(0))
    assert np.all(orc.attention(q, k[:1], v[:1], 2, 0.125)[0][0] == 0)      # the first of two rows sees none of one key


def cache(heads=2, D=128, P=64, pages=4, data=0x10000):
    return qa.KvQ4(heads, D, P, pages, data)


def store(c, T=1, k=0x1000, nbk=None, v=0x2000, nbv=None, slot=0x3000, typ=qa.F32, fn="qwmoe_kv_q4_store"):
    nb = 2 * 128 * 4
    return getattr(qa.lib(), fn)(None, C.byref(c) if c is not None else None, typ, k, nb if nbk is None else nbk, v,
                                 nb if nbv is None else nbv, slot, T)


@pytest.mark.parametrize("fn", ["qwmoe_kv_q4_store", "qwmoe_kv_q4_load"])
def test_rows_refusals(fn):
    assert store(None, fn=fn) == INVALID
    for c in (cache(heads=0), cache(P=0), cache(pages=0), cache(data=None), cache(D=0), cache(heads=-1)):
        assert store(c, fn=fn) == INVALID
    for c in (cache(D=96), cache(D=512), cache(P=48), cache(P=16), cache(P=8192), cache(data=0x10008), cache(pages=1 << 31)):
        assert store(c, fn=fn) == UNSUPPORTED
    for kw in ({"k": None}, {"v": None}, {"slot": None}, {"T": -1}, {"nbk": 1008}, {"nbv": 0}):
        assert store(cache(), fn=fn, **kw) == INVALID
    for kw in ({"typ": qa.Q8_0}, {"typ": qa.I32}, {"k": 0x1004}, {"v": 0x2008}, {"nbk": 1028}, {"nbv": 1032}):
        assert store(cache(), fn=fn, **kw) == UNSUPPORTED
    assert store(cache(), fn=fn) == NOT_READY


def plan(**kw):
    a = dict(held=0x100, past=0x200, new=0x300, S=4, P=64, N=100, table=0x400, W=8, ring=0x500, counters=0x600, out=0x700, T=4,
             start=0x800, lens=0x900, slot=0xA00, pos=0xB00)
    a.update(kw)
    return qa.lib().qwmoe_kv_plan(None, a["held"], a["past"], a["new"], a["S"], a["P"], a["N"], a["table"], a["W"], a["ring"],
                                  a["counters"], a["out"], a["T"], a["start"], a["lens"], a["slot"], a["pos"])


def test_plan_refusals():
    for name in ("held", "past", "new", "table", "ring", "counters", "out", "start", "lens", "slot", "pos"):
        assert plan(**{name: None}) == INVALID, name
    for kw in ({"S": 0}, {"S": -1}, {"N": 0}, {"W": 0}, {"T": -1}, {"P": 0}, {"out": 0x600}):
        assert plan(**kw) == INVALID, kw
    for kw in ({"S": 4097}, {"P": 33}, {"P": 16}, {"P": 8192}, {"N": 1 << 31}, {"T": 1 << 31}, {"W": 1 << 25}):
        assert plan(**kw) == UNSUPPORTED, kw
    assert plan() == NOT_READY
    assert plan(T=0, slot=None, pos=None) == NOT_READY


def attn(c=None, **kw):
    a = dict(typ=qa.F32, q=0x1000, nbq=8 * 512, nq=8, table=0x100, W=8, start=0x200, lens=0x300, S=4, T=4, max_new=1, max_len=512,
             scale=0.0, out=0x8000, nbo=8 * 512)
    a.update(kw)
    c = cache() if c is None else c
    return qa.lib().qwmoe_attn_kv_q4(None, C.byref(c), a["typ"], a["q"], a["nbq"], a["nq"], a["table"], a["W"], a["start"],
                                     a["lens"], a["S"], a["T"], a["max_new"], a["max_len"], a["scale"], a["out"], a["nbo"])


def test_attention_refusals():
    for name in ("q", "table", "start", "lens", "out"):
        assert attn(**{name: None}) == INVALID, name
    for kw in ({"nq": 0}, {"nq": 7}, {"W": 0}, {"S": 0}, {"T": -1}, {"max_new": -1}, {"max_len": -1}, {"max_len": 513},
               {"out": 0x1000}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"nbq": 4080}, {"nbo": 16}):
        assert attn(**kw) == INVALID, kw
    for kw in ({"typ": qa.Q4_K}, {"S": 4097}, {"nq": 65538}, {"W": 1 << 25}, {"T": 1 << 30}, {"q": 0x1008}, {"out": 0x8004},
               {"nbq": 4104}, {"nbo": 4100}):
        assert attn(**kw) == UNSUPPORTED, kw
    assert attn(cache(D=96)) == UNSUPPORTED and attn(cache(P=40)) == UNSUPPORTED
    assert attn() == NOT_READY


def test_page_bytes():
    f = qa.lib().qwmoe_kv_q4_page_bytes
    assert f(4, 128, 64) == 4 * 2 * 36 * 128 and f(1, 256, 32) == 36 * 256
    assert f(0, 128, 64) == 0 and f(4, 100, 64) == 0 and f(4, 128, 100) == 0 and f(4, 128, 16) == 0


def test_wrapper_refusals():
    torch = pytest.importorskip("torch")
    from questwend_amd import ops
    size = ops.kv_q4_page_bytes(2, 64, 32)
    data = torch.zeros(3 * size, dtype=torch.uint8)
    c = ops.make_kv_q4(data, 2, 64, 32)
    assert c.n_pages == 3
    for bad in (data[:-1], data.view(torch.int8), data[:0]):
        with pytest.raises(ValueError):
            ops.make_kv_q4(bad, 2, 64, 32)
    with pytest.raises(ValueError):
        ops.make_kv_q4(data, 2, 65, 32)
    slot = torch.zeros(4, dtype=torch.int64)
    k = torch.zeros(4, 2, 64)
    with pytest.raises(TypeError):
        ops.kv_q4_store(c, k.double(), k.double(), slot)
    for kk, vv, ss in ((k[:, :1], k, slot), (k, k.half(), slot), (k, k[:3], slot), (k, k, slot.int()), (k, k, slot[:3]),
                       (k.transpose(1, 2).contiguous().transpose(1, 2), k, slot)):
        with pytest.raises(ValueError):
            ops.kv_q4_store(c, kk, vv, ss)
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        ops.attn_kv_q4(c, torch.zeros(4, 6, 64), i32(2, 3), i32(2), i32(2), 1, 64)
    with pytest.raises(ValueError):
        ops.attn_kv_q4(c, torch.zeros(4, 6, 32), i32(2, 3), i32(3), i32(2), 1, 64)
    with pytest.raises(ValueError):
        ops.kv_plan(i32(2), i32(2), i32(3), 32, i32(2, 3), i32(9), torch.zeros(2, dtype=torch.int64), 4)


def test_scale_range():
    for scale in (2.0**-20, 2.0**20, 0.0, 0.125):
        assert attn(scale=scale) == NOT_READY
    for scale in (2.0**-21, 2.0**21, 1e-40, 1e30):
        assert attn(scale=scale) == UNSUPPORTED


def test_wrappers_refuse_other_devices(monkeypatch):
    """Tensors that are not the current device's never reach a kernel (here: host tensors)."""
    torch = pytest.importorskip("torch")
    from questwend_amd import ops
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    c = ops.make_kv_q4(torch.zeros(3 * ops.kv_q4_page_bytes(2, 64, 32), dtype=torch.uint8), 2, 64, 32)
    k, slot = torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int64)
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    for call in (lambda: ops.kv_q4_store(c, k, k, slot), lambda: ops.kv_q4_load(c, slot),
                 lambda: ops.attn_kv_q4(c, torch.zeros(4, 6, 64), i32(2, 3), i32(3), i32(2), 1, 64),
                 lambda: ops.kv_plan(i32(2), i32(2), i32(2), 32, i32(2, 3), i32(9), torch.zeros(2, dtype=torch.int64), 4)):
        with pytest.raises(ValueError, match="current device"):
            call()
