"""GPU checks of the paged 4-bit cache (qwmoe_kv_plan, qwmoe_kv_q4_store, qwmoe_kv_q4_load,
qwmoe_attn_kv_q4) against kv_q4_oracle's definitions in 64 bits.

Pools start as 0xFF bytes (every scale a NaN), so anything read beyond a request's
tokens shows.  The bookkeeping and the stored bytes are compared exactly; read rows to
half a step of their type; attention to a bound derived from its roundings:

  scores    products and sums of D terms in fp32, an f32 q in two f16 parts (2^-22 each
            product), scaling and the exponential's argument: at most
            delta = B ((D + 16) 2^-24 + 2^-21), B = max_j sum |q k_j| scale;
  weights   2 delta, exp2 and the sums over len keys: (len + 64) 2^-24 + 2^-21; f16 and bf16
            rows round each weight to f16: 2^-11; weights far below the largest are
            f16 subnormals: 2^-28 of it each;
  bf16      requests of many rows: keys and values rounded once to f16, 2^-11 each (B 2^-11 in delta);
  values    all of it times sum p |v| (and len max |v| for the last), the codes being exact;
  output    half a step of its type.
"""
from __future__ import annotations

import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import kv_q4_oracle as orc  # noqa: E402
import questwend_amd as qa  # noqa: E402
from questwend_amd import ops  # noqa: E402

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def note(msg: str) -> None:
    print(f"[gpu-kv-q4] {msg}", flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module", autouse=True)
def lib_init():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    ops.init(0, 512 << 20)
    ops.device_status(clear=True)
    yield
    torch.cuda.synchronize()


@pytest.fixture(autouse=True)
def named(request):
    note(request.node.name)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    return t if dtype is None else t.to(dtype)


def i32(a):
    return dev(np.asarray(a, np.int32))


def rows(rng, shape, dtype, std=1.0):
    """Random rows on the GPU and, exactly, in f64."""
    t = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(DEV).to(dtype)
    return t, t.double().cpu().numpy()


def new_cache(n_pages, heads, D, P):
    data = torch.full((n_pages * ops.kv_q4_page_bytes(heads, D, P),), 0xFF, dtype=torch.uint8, device=DEV)
    return ops.make_kv_q4(data, heads, D, P), data


def status():
    return ops.device_status(clear=True)


# ---- rows ----------------------------------------------------------------------


@pytest.mark.parametrize("D,heads,P", [(128, 4, 64), (64, 3, 32), (256, 2, 128), (128, 1, 256)])
@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("T", [1, 3, 37, 130])
def test_store_bytes(D, heads, P, typ, T):
    rng = np.random.default_rng(D + heads + T)
    pages = 5
    cache, data = new_cache(pages, heads, D, P)
    want = orc.Cache(pages, heads, D, P)
    slots = rng.permutation(pages * P)[:T].astype(np.int64)
    if T == 37:                                   # consecutive slots from an odd place on
        slots = np.arange(T) + 13
    if T == 130:
        slots = np.concatenate([np.arange(90) + 5, slots[~np.isin(slots, np.arange(90) + 5)]])[:T]
        slots = np.concatenate([slots, rng.permutation(np.setdiff1d(np.arange(pages * P), slots))])[:T]
        slots[[7, 50]] = -1
    k, k64 = rows(rng, (T, heads, D), TYPES[typ])
    v, v64 = rows(rng, (T, heads, D), TYPES[typ], 0.3)
    ops.kv_q4_store(cache, k, v, dev(slots))
    want.store(k64, v64, slots)
    assert np.array_equal(data.cpu().numpy(), want.data)
    ok = slots >= 0
    if ok.all():
        got = ops.kv_q4_load(cache, dev(slots), TYPES[typ])
        for g, w in zip(got, want.load(slots)):
            assert torch.equal(g.cpu(), torch.from_numpy(w).to(TYPES[typ]))   # (one rounding of the exact value)
    assert status() == 0


def test_store_strided_rows_and_edges():
    rng = np.random.default_rng(5)
    D, heads, P, T = 128, 2, 32, 24
    cache, data = new_cache(3, heads, D, P)
    want = orc.Cache(3, heads, D, P)
    wide = torch.from_numpy(rng.standard_normal((T, 5 * heads * D)).astype(np.float32)).to(DEV)
    k = wide[:, heads * D:2 * heads * D].view(T, heads, D)
    v = wide[:, 3 * heads * D:4 * heads * D].view(T, heads, D)
    k[0, 0, 5], k[1, 0, 40], k[2, 1, 100], k[3, 0, 0] = float("inf"), float("nan"), -float("inf"), 3e38
    k[4] = 0.0
    v[5, 1, :32] = 1e-9
    v[6, 0, 32:34] = torch.tensor([4.0, -4.0], device=DEV)
    v[7] = -0.0
    v[8, 0] *= 1e-7                              # subnormal scales
    for s in range(16):                          # values on the borders between codes
        v[9, 1, s] = (s - 7.5) * 0.25
    v[9, 1, 16:32] = -2.0
    slots = rng.permutation(3 * P)[:T]
    ops.kv_q4_store(cache, k, v, dev(slots))
    want.store(k.double().cpu().numpy(), v.double().cpu().numpy(), slots)
    a, b = data.cpu().numpy(), want.data
    # a NaN scale is a NaN, whatever its bits; its block's codes are the middle one
    got = ops.kv_q4_load(cache, dev(slots))
    for g, w in zip(got, want.load(slots)):
        assert np.array_equal(g.cpu().numpy().astype(np.float64), w, equal_nan=True)
    differ = np.nonzero(a != b)[0]
    assert len(differ) <= 2 * 3, "bytes beyond the three NaN scales differ"
    assert status() == 0


@pytest.mark.parametrize("bad", [3 * 64, 1 << 40, (1 << 62) + 5])
def test_slots_outside_the_pool(bad):
    cache, data = new_cache(3, 2, 64, 64)
    k = torch.ones(4, 2, 64, device=DEV)
    ops.kv_q4_store(cache, k, k, dev(np.array([bad, -1, 70, -(1 << 60)])))
    assert status() == qa.STATUS_BAD_SLOT
    want = orc.Cache(3, 2, 64, 64)
    want.store(np.ones((1, 2, 64)), np.ones((1, 2, 64)), [70])
    assert np.array_equal(data.cpu().numpy(), want.data)
    out = (torch.full((4, 2, 64), 9.0, device=DEV), torch.full((4, 2, 64), 9.0, device=DEV))
    ops.kv_q4_load(cache, dev(np.array([70, bad, -1, 70])), out=out)
    assert status() == qa.STATUS_BAD_SLOT
    for o in out:
        assert torch.equal(o[:, 0, 0].cpu(), torch.tensor([1.0, 9.0, 9.0, 1.0]))


@pytest.mark.parametrize("typ", list(TYPES))
def test_load_repeats_and_strides(typ):
    rng = np.random.default_rng(8)
    D, heads, P = 64, 3, 32
    cache, data = new_cache(4, heads, D, P)
    every = np.arange(4 * P)
    k, _ = rows(rng, (4 * P, heads, D), torch.float32)
    v, _ = rows(rng, (4 * P, heads, D), torch.float32, 50.0)
    ops.kv_q4_store(cache, k, v, dev(every))
    ref = orc.Cache(4, heads, D, P)
    ref.data = data.cpu().numpy()
    slots = rng.integers(0, 4 * P, 61)
    slots[3:8] = 17
    slots[10] = -1
    buf = torch.full((61, 4, heads, D), 7.0, device=DEV, dtype=TYPES[typ])
    ops.kv_q4_load(cache, dev(slots), out=(buf[:, 1], buf[:, 3]))
    for j, w in zip((1, 3), ref.load(np.maximum(slots, 0))):
        w = torch.from_numpy(w).to(TYPES[typ])
        w[10] = 7.0
        assert torch.equal(buf[:, j].cpu(), w)
    assert torch.equal(buf[:, 0], torch.full_like(buf[:, 0], 7.0)) and torch.equal(buf[:, 2], torch.full_like(buf[:, 2], 7.0))


# ---- bookkeeping -----------------------------------------------------------------


def run_plan(held, past, new, P, table, ring, counters, T):
    t, r = i32(table), i32(ring)
    got = ops.kv_plan(i32(held), i32(past), i32(new), P, t, r, dev(np.asarray(counters, np.int64)), T)
    return t.cpu().numpy(), r.cpu().numpy(), [x.cpu().numpy() for x in got], status()


def check_plan(held, past, new, P, table, ring, counters, T):
    wt, wr = table.copy(), ring.copy()
    want = orc.plan(held, past, new, P, wt, wr, counters, T)
    gt, gr, got, st = run_plan(held, past, new, P, table, ring, counters, T)
    for g, w, name in zip(got, want, ("counters", "seq_start", "seq_len", "slot", "pos")):
        assert np.array_equal(g, w), name
    assert np.array_equal(gt, wt), "page_table"
    assert np.array_equal(gr, wr), "ring"
    assert st == want[5]
    return wt, wr, want


@pytest.mark.parametrize("S", [1, 2, 63, 64, 65, 255, 256, 257, 700, 4096])
@pytest.mark.parametrize("P", [32, 64, 4096])
def test_plan_rounds(S, P):
    """Several rounds of one batch: growth, shrinking, ends, idle requests, a ring that goes round."""
    rng = np.random.default_rng(S + P)
    W = 6
    n_pages = max(3, 2 * S + 1)
    table = np.full((S, W), -7, np.int32)
    ring = rng.permutation(n_pages).astype(np.int32)
    counters = np.array([11 * n_pages + 3, 12 * n_pages + 3])
    held = np.zeros(S, np.int64)
    lacked = False
    for step in range(5):
        past = np.where(rng.random(S) < 0.2, 0, np.maximum(held - rng.integers(0, 40, S), 0))
        new = np.where(rng.random(S) < 0.3, 0, rng.integers(0, max(2, min(3 * P, 200)), S))
        new = np.minimum(new, W * P - past)
        T = int(new.sum()) + (step % 2) * 5
        table, ring, want = check_plan(held, past, new, P, table, ring, counters, T)
        counters = want[0]
        served = (want[2] > 0) | (past + new == 0)
        lacked |= bool(want[5] & 16)
        held = np.where(served, past + new, held)
        used = [table[i, c] for i in range(S) for c in range(-(-int(held[i]) // P))]
        free = [ring[x % n_pages] for x in range(counters[0], counters[1])]
        assert sorted(used + free) == list(range(n_pages)), "pages lost or doubled"
    assert lacked or P == 4096 or S < 3


def test_plan_bad_lengths_and_rows():
    n_pages, P, W = 40, 32, 4
    table = np.arange(9 * W, dtype=np.int32).reshape(9, W)
    ring = np.full(n_pages, -1, np.int32)
    ring[:4] = [36, 37, 38, 39]
    #       fine  neg new  neg past  past > held  too wide  neg held  fine  rows behind T  fine: 0 rows
    held = [10,   10,      10,       10,          10,       -5,       33,   5,             64]
    past = [10,   10,      -3,       11,          10,       0,        33,   5,             20]
    new = [30,    -4,      2,        2,           125,      3,        1,    50,            0]
    check_plan(held, past, new, P, table, ring, np.array([0, 4]), 10 ** 3)
    check_plan(held, past, new, P, table, ring, np.array([0, 4]), 170)
    check_plan(held, past, new, P, table, ring, np.array([0, 4]), 0)
    check_plan([0x7fffffff], [0x7fffffff], [0x7fffffff], P, table[:1], ring, np.array([0, 4]), 5)
    check_plan([0] * 3, [0] * 3, [3, 0x7fffffff, 3], P, table[:3], ring, np.array([0, 4]), 5)


def test_plan_pages_outside_the_pool_and_odd_counters():
    table = np.array([[99, 2, 3], [-1, 0, 0], [5, 1, 1]], np.int32)
    ring = np.array([7, 8, -9, 3, 4, 5, 6, 0, 1, 2], np.int32)
    check_plan([40, 20, 0], [40, 20, 0], [30, 3, 70], 32, table, ring, np.array([1, 4]), 120)
    check_plan([0], [0], [3], 32, table[:1], ring, np.array([5, 5]), 3)          # nothing free
    check_plan([0], [0], [3], 32, table[:1], ring, np.array([9, 5]), 3)          # a tail before its head
    check_plan([0], [0], [3], 32, table[:1], ring, np.array([-13, -10]), 3)      # counters below zero


# ---- attention -------------------------------------------------------------------


class Batch:
    """Requests with their rows in a pool of scattered pages."""

    def __init__(self, seed, heads, D, P, lens, new, typ, Hq, kstd=1.0, vstd=0.5, qstd=2.0, kmul=None, vmul=None, pad=0, spare=1):
        rng = np.random.default_rng(seed)
        self.lens, self.new, self.typ, self.Hq, self.D, self.P = lens, new, TYPES[typ], Hq, D, P
        need = [-(-n // P) for n in lens]
        n_pages = sum(need) + spare
        perm = rng.permutation(n_pages)
        W = max(need + [1]) + 1
        self.table = np.full((len(lens), W), 0x7fffffff, np.int64)     # entries behind a request's pages are never used
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        self.table = self.table.astype(np.int32)
        self.cache, self.data = new_cache(n_pages, heads, D, P)
        self.k64, self.v64 = [], []
        for i, n in enumerate(lens):
            k = (rng.standard_normal((n, heads, D)) * kstd).astype(np.float32)
            v = (rng.standard_normal((n, heads, D)) * vstd).astype(np.float32)
            if kmul is not None:
                k *= kmul(np.arange(n), n)[:, None, None].astype(np.float32)
            if vmul is not None:
                v *= vmul(np.arange(n), n)[:, None, None].astype(np.float32)
            if n:
                ops.kv_q4_store(self.cache, dev(k), dev(v), dev(self.slots(i, np.arange(n))))
            self.k64.append(orc.values(*orc.quantize(k)) if n else np.zeros((0, heads, D)))
            self.v64.append(orc.values(*orc.quantize(v)) if n else np.zeros((0, heads, D)))
        self.start = np.concatenate([[0], np.cumsum(new)])
        self.T = int(self.start[-1]) + pad
        self.q, self.q64 = rows(rng, (self.T, Hq, D), self.typ, qstd)

    def slots(self, i, pos):
        return self.table[i, pos // self.P].astype(np.int64) * self.P + pos % self.P

    def run(self, q=None, out=None, max_new=None, max_len=None, scale=0.0):
        return ops.attn_kv_q4(self.cache, self.q if q is None else q, dev(self.table), i32(self.start), i32(self.lens),
                              max(list(self.new) + [1]) if max_new is None else max_new,
                              max(list(self.lens) + [1]) if max_len is None else max_len, scale, out)

    def check(self, got, scale=None, requests=None, but=()):
        """Every row against the oracle; but: (row, heads) to pass over."""
        scale = self.D ** -0.5 if scale is None else scale
        for i, (n, length) in enumerate(zip(self.new, self.lens)):
            if not n or (requests is not None and i not in requests):
                continue
            a = int(self.start[i])
            g = got[a:a + n].double().cpu().numpy()
            want, mag, big = orc.attention(self.q64[a:a + n], self.k64[i], self.v64[i], n, scale)
            bf16 = 2.0**-11 if self.typ == torch.bfloat16 else 0.0
            delta = big * ((self.D + 16) * 2.0**-24 + 2.0**-21 + bf16)
            tol = mag * (2 * delta * (1 + delta) + (length + 64) * 2.0**-24 + 2.0**-21 + (0 if self.typ == torch.float32 else 2.0**-11) + bf16)
            vmax = np.abs(self.v64[i]).max() if length else 0.0
            tol = tol + length * vmax * 2.0**-28 + np.abs(want) * (torch.finfo(self.typ).eps / 2) + 2.0**-25
            for r, heads in but:
                if a <= r < a + n:
                    g[r - a, heads] = want[r - a, heads]
            off = np.abs(g - want)
            assert np.all(np.isfinite(g)), f"request {i}: not finite"
            worst = float((off / tol).max())
            assert worst <= 1, f"request {i} (len {length}, new {n}): {worst:.3g} of the bound, {float(off.max()):.3g} off"


HEADS = [(128, 4, 32), (128, 2, 8), (64, 2, 14), (256, 2, 16), (128, 3, 3), (64, 1, 20)]
LENS = [([1], [1]), ([31, 32, 33, 64, 65], [1] * 5), ([700], [1]), ([257, 5, 1000, 40], [5, 5, 5, 5]),
        ([130], [130]), ([300, 64, 2, 129], [33, 1, 2, 100]), ([513, 96], [200, 0])]


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("D,heads,Hq", HEADS)
@pytest.mark.parametrize("case", range(len(LENS)))
def test_attention(typ, D, heads, Hq, case):
    lens, new = LENS[case]
    P = [64, 32, 128, 64, 32, 256, 4096][(case + heads) % 7]
    b = Batch(case * 10 + D, heads, D, P, lens, new, typ, Hq)
    b.check(b.run())
    assert status() == 0


@pytest.mark.parametrize("typ", list(TYPES))
def test_attention_empty_rows_and_padding(typ):
    b = Batch(3, 2, 128, 32, [0, 40, 3, 0, 70], [2, 1, 5, 0, 4], typ, 8, pad=6)
    out = torch.full_like(b.q, 5.0)
    b.run(out=out)
    assert torch.equal(out[b.start[-1]:], torch.full_like(out[b.start[-1]:], 5.0)), "rows behind the last request"
    assert torch.count_nonzero(out[:2]) == 0, "a request without keys"
    assert torch.count_nonzero(out[3:5]) == 0, "the rows of a request with more new tokens than keys"
    b.check(out)
    assert status() == 0
    for T in (0,):
        q = b.q[:T]
        assert ops.attn_kv_q4(b.cache, q, dev(b.table), i32([0] * 6), i32(b.lens), 5, 70).shape[0] == 0


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("D,heads,Hq", [(128, 2, 8), (256, 1, 4)])
@pytest.mark.parametrize("shape", ["tiny", "huge", "rising", "falling", "mixed", "steep", "peaked"])
def test_attention_ranges(typ, D, heads, Hq, shape):
    """Values over f16's scales, up and down along the keys; scores that keep rising; one key far above all."""
    vmul = {"tiny": lambda i, n: np.full(n, 1e-3), "huge": lambda i, n: np.full(n, 1e3),
            "rising": lambda i, n: 10.0 ** (-3 + 6 * i / n), "falling": lambda i, n: 10.0 ** (3 - 6 * i / n),
            "mixed": lambda i, n: 10.0 ** ((i * 7919) % 6 - 3.0)}.get(shape)
    kmul = {"steep": lambda i, n: 0.1 + 4.0 * i / n, "peaked": lambda i, n: np.where(i == n // 2, 20.0, 0.05)}.get(shape)
    for lens, new in (([301], [1]), ([150, 520], [40, 3])):
        b = Batch(D + len(shape), heads, D, 64, lens, new, typ, Hq, kmul=kmul, vmul=vmul)
        b.check(b.run())
    assert status() == 0


@pytest.mark.parametrize("typ", list(TYPES))
def test_attention_scores_far_below(typ):
    """Every score hundreds below zero, all the same key, and a scale that is given."""
    b = Batch(9, 1, 64, 32, [77], [3], typ, 2, kstd=0.0, kmul=lambda i, n: np.ones(n))
    k = np.full((77, 1, 64), -3.0, np.float32)
    ops.kv_q4_store(b.cache, dev(k), torch.zeros(77, 1, 64, device=DEV) + 0.25, dev(b.slots(0, np.arange(77))))
    b.k64[0], b.v64[0] = orc.values(*orc.quantize(k)), np.full((77, 1, 64), 0.25)
    b.q.fill_(3.0)
    b.q64 = np.full_like(b.q64, 3.0)
    b.check(b.run(scale=1.0), scale=1.0)


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_attention_nan_stays_where_it_is_seen(typ, new):
    b = Batch(4, 2, 128, 32, [150, 90], new, typ, 8)
    clean = b.run()
    b.check(clean)
    # request 0's last key and value hold NaN and infinity: only the rows that see them change
    k, v = torch.randn(1, 2, 128, device=DEV), torch.randn(1, 2, 128, device=DEV)
    k[0, 0, 7], v[0, 1, 100] = float("nan"), float("inf")
    ops.kv_q4_store(b.cache, k, v, dev(b.slots(0, np.array([149]))))
    got = b.run()
    n = new[0]
    # Rows that do not see the new key keep their values to the bound, not to the bit: the bound 2^E of the value
    # scales is one for a wave's rows, and where it moves, the weights' exponents s - off are rounded anew (off, an
    # integer further on, has other last bits).  The other request's rows are other waves'.
    b.check(got, but=[(n - 1, slice(None))])
    assert torch.equal(got[n:], clean[n:])
    assert torch.isnan(got[n - 1, :4]).all()                                   # kv head 0: a NaN score
    v1 = got[n - 1, 4:]
    assert torch.isnan(v1[:, 96:128]).all() and torch.isfinite(v1[:, :96]).all()   # kv head 1: one block of values
    # a NaN or an infinity in q stays in its row (an infinite score sets the others' offsets anew, as above)
    q = b.q.clone()
    q[0, 3, 64], q[n, 6, 0] = float("nan"), float("inf")
    got = b.run(q=q)
    assert torch.isnan(got[0, 3]).all() and torch.isnan(got[n, 6]).all()
    b.check(got, but=[(n - 1, slice(None)), (0, 3), (n, 6)])
    assert status() == 0


def test_attention_beyond_the_bounds():
    b = Batch(6, 2, 64, 32, [100, 50, 64], [3, 2, 4], "f32", 4)
    clean = b.run()
    got = b.run(max_len=64)
    assert status() == qa.STATUS_BAD_SEQ
    assert torch.count_nonzero(got[:3]) == 0
    b.check(got, requests=[1, 2])
    got = b.run(max_new=3)
    assert status() == qa.STATUS_BAD_SEQ
    assert torch.count_nonzero(got[5:]) == 0
    b.check(got, requests=[0, 1])
    b.lens[1] = -4
    got = b.run()
    assert status() == qa.STATUS_BAD_SEQ and torch.count_nonzero(got[3:5]) == 0
    b.lens[1] = 50
    # a page outside the pool: its keys count as masked, the request's others as they are
    keep = b.table[0].copy()
    for wrong in (-1, b.cache.n_pages, 0x7fffffff):
        b.table[0, 1] = wrong
        got = b.run()
        assert status() == qa.STATUS_BAD_SLOT
        k, v = b.k64[0], b.v64[0]
        seen = np.r_[0:32, 64:100]
        b.k64[0], b.v64[0], b.lens[0] = k[seen], v[seen], 68
        b.check(got)
        b.k64[0], b.v64[0], b.lens[0] = k, v, 100
    b.table[0] = keep
    assert torch.equal(b.run(), clean)
    assert status() == 0


def test_attention_strided_rows():
    b = Batch(12, 2, 128, 64, [90, 33], [20, 1], "bf16", 8)
    wide = torch.full((b.T, 3, 8, 128), 2.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 1] = b.q
    out = torch.full((b.T, 2, 8, 128), 4.0, dtype=torch.bfloat16, device=DEV)
    b.run(q=wide[:, 1], out=out[:, 1])
    assert torch.equal(out[:, 1], b.run())
    assert torch.equal(out[:, 0], torch.full_like(out[:, 0], 4.0))
    b.check(out[:, 1])


@pytest.mark.parametrize("typ,length", [("f32", 40000), ("bf16", 30011)])
def test_attention_long(typ, length):
    b = Batch(20, 1, 128, 256, [length, 17], [1, 1], typ, 8)
    b.check(b.run())
    # a bound far above the lengths changes the split, not the result beyond rounding
    wide = np.full((2, 4096), 0x7fffffff, np.int32)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide
    b.check(b.run(max_len=1 << 20, max_new=9))
    assert status() == 0


def test_attention_small_workspace_shares_the_long_axis():
    """Whatever the workspace holds, the call gives its result (fewer splits where it holds fewer)."""
    b = Batch(21, 1, 128, 64, [6000, 3000], [1, 2], "f32", 8)
    try:
        torch.cuda.synchronize()
        ops.shutdown()
        ops.init(0, 40 << 10)
        b.check(b.run())
        ops.shutdown()
        ops.init(0, 1 << 10)
        b.check(b.run())
    finally:
        torch.cuda.synchronize()
        ops.shutdown()
        ops.init(0, 512 << 20)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB: rows stored, read and attended to in its last pages."""
    heads, D, P, length = 8, 256, 4096, 5000
    size = ops.kv_q4_page_bytes(heads, D, P)
    n_pages = (5 << 30) // size
    data = torch.empty(n_pages * size, dtype=torch.uint8, device=DEV)
    b = Batch(30, heads, D, P, [4097], [2], "f16", 8, spare=0)
    b.cache = ops.make_kv_q4(data, heads, D, P)
    b.table = np.array([[n_pages - 1, n_pages - 2]], np.int32)
    rng = np.random.default_rng(1)
    k = rng.standard_normal((4097, heads, D)).astype(np.float32)
    v = rng.standard_normal((4097, heads, D)).astype(np.float32)
    slots = dev(b.slots(0, np.arange(4097)))
    ops.kv_q4_store(b.cache, dev(k), dev(v), slots)
    b.k64, b.v64 = [orc.values(*orc.quantize(k))], [orc.values(*orc.quantize(v))]
    for g, w in zip(ops.kv_q4_load(b.cache, slots), (b.k64[0], b.v64[0])):
        assert np.array_equal(g.cpu().numpy().astype(np.float64), w)
    b.check(b.run())
    assert status() == 0


# ---- as they are used ---------------------------------------------------------------


def generate(graph: bool, typ: str):
    """A server's life: three requests' prompts, decode and draft steps with rejections, an end, a new request; every
    step plan -> store -> attention, eager or through one captured graph of fixed sizes.  Returns every step's outputs."""
    rng = np.random.default_rng(77)
    heads, Hq, D, P, S, W, T, n_pages = 2, 8, 128, 32, 4, 8, 60, 20
    cache, data = new_cache(n_pages, heads, D, P)
    table = torch.zeros((S, W), dtype=torch.int32, device=DEV)
    ring = i32(rng.permutation(n_pages))
    counters = dev(np.array([0, n_pages]))
    held, past, new = (torch.zeros(S, dtype=torch.int32, device=DEV) for _ in range(3))
    q = torch.zeros((T, Hq, D), dtype=TYPES[typ], device=DEV)
    k, v = (torch.zeros((T, heads, D), dtype=TYPES[typ], device=DEV) for _ in range(2))
    out = torch.zeros_like(q)
    state = {}

    def step():
        nxt, start, lens, slot, pos = ops.kv_plan(held, past, new, P, table, ring, counters, T)
        ops.kv_q4_store(cache, k, v, slot)
        ops.attn_kv_q4(cache, q, table, start, lens, 40, W * P, out=out)
        counters.copy_(nxt)
        state.update(start=start, lens=lens, slot=slot, pos=pos)

    #          prompts           decode          drafts        2 rejected, 1 ends   prompt of a new one    decode
    plans = [([0, 0, 0, 0], [33, 20, 5, 0]), (None, [1, 1, 1, 0]), (None, [5, 5, 5, 0]), ([-3, 0, -5, 0], [1, 0, 4, 30]),
             (None, [1, 40, 1, 1]), (None, [1, 1, 1, 1]), (None, [1, 1, 1, 1])]
    g = None
    results, length = [], np.zeros(S, np.int64)
    hist = [[np.zeros((0, heads, D)), np.zeros((0, heads, D))] for _ in range(S)]
    for at, (drop, n) in enumerate(plans):
        p = length + (np.array(drop) if drop and at else 0)
        if at == 3:
            p[1] = 0
        held.copy_(i32(length)), past.copy_(i32(p)), new.copy_(i32(n))
        for x, std in ((q, 2.0), (k, 1.0), (v, 0.5)):
            x.copy_(torch.from_numpy((rng.standard_normal(tuple(x.shape)) * std).astype(np.float32)))
        out.fill_(3.0)
        if not graph:
            step()
        else:
            if g is None:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    step()
            torch.cuda.synchronize()
            g.replay()
            (torch.randn(1000, device=DEV) ** 2).sum().item()      # the program's own work between the replays
        torch.cuda.synchronize()
        start = np.concatenate([[0], np.cumsum(n)])
        assert np.array_equal(state["start"].cpu().numpy(), start) and np.array_equal(state["lens"].cpu().numpy(), p + n)
        k64, v64, q64 = (x.double().cpu().numpy() for x in (k, v, q))
        for i in range(S):
            for j, x in enumerate((k64, v64)):
                hist[i][j] = np.concatenate([hist[i][j][:p[i]], orc.values(*orc.quantize(x[start[i]:start[i + 1]]))])
            if n[i]:
                want, mag, big = orc.attention(q64[start[i]:start[i + 1]], *hist[i], n[i], D ** -0.5)
                got = out[start[i]:start[i + 1]].double().cpu().numpy()
                tol = mag * (2.0**-10 if typ != "f32" else 2.0**-14) + np.abs(want) * torch.finfo(TYPES[typ]).eps
                assert np.all(np.abs(got - want) <= tol + 2.0**-20), (at, i)
        assert torch.equal(out[start[-1]:], torch.full_like(out[start[-1]:], 3.0))
        length = p + n
        results.append(out.clone())
    assert status() == 0
    return results


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_plan_store_attention_together(typ):
    eager = generate(False, typ)
    replayed = generate(True, typ)
    for a, b in zip(eager, replayed):
        assert torch.equal(a, b)


def test_other_stream_and_two_graphs_on_one_workspace():
    a = Batch(40, 1, 128, 64, [3000], [1], "f32", 8)
    b = Batch(41, 1, 128, 64, [2500, 900], [2, 1], "f16", 4)
    wa, wb = a.run(), b.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = a.run()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, wa)
    outs, graphs = [torch.zeros_like(wa), torch.zeros_like(wb)], []
    for x, o in ((a, outs[0]), (b, outs[1])):
        args = (dev(x.table), i32(x.start), i32(x.lens))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.attn_kv_q4(x.cache, x.q, *args, max(x.new), max(x.lens), out=o)
        graphs.append((g, args))
    for _ in range(4):
        for o in outs:
            o.zero_()
        for g, _ in graphs:
            g.replay()
        assert torch.equal(a.run(), wa)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wa) and torch.equal(outs[1], wb)
    assert status() == 0


def test_same_call_twice_gives_the_same_bits():
    b = Batch(50, 2, 128, 64, [5000, 100, 1200], [1, 20, 5], "f32", 16)
    first = b.run()
    for _ in range(5):
        assert torch.equal(b.run(), first)


# ---- requests of many rows: the keys split over workgroups -----------------------------


MANY = [(128, 1, 8, 64), (64, 2, 14, 128), (256, 1, 8, 32), (128, 2, 2, 256)]


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("D,heads,Hq,P", MANY)
@pytest.mark.parametrize("lens,new", [([3000], [140]), ([2500, 700, 60], [150, 1, 3]), ([129, 1900], [129, 200])])
def test_many_rows_over_splits(typ, D, heads, Hq, P, lens, new):
    b = Batch(60 + D, heads, D, P, lens, new, typ, Hq, pad=3)
    out = torch.full_like(b.q, 5.0)
    b.run(out=out)
    b.check(out)
    assert torch.equal(out[b.start[-1]:], torch.full_like(out[b.start[-1]:], 5.0))
    b.check(b.run(max_new=max(new) + 77, max_len=b.table.shape[1] * P))       # wider bounds: other splits
    assert status() == 0


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("D,heads,Hq,P", MANY)
def test_many_rows_bad_pages_and_nans(typ, D, heads, Hq, P):
    """A page outside the pool in the middle of the keys, and a NaN and an infinity that only the last row sees."""
    n, new = 2000, 150
    b = Batch(61, heads, D, P, [n], [new], typ, Hq)
    keep, at = b.table.copy(), 1000 // P
    b.table[0, at] = b.cache.n_pages
    got = b.run()
    assert status() == qa.STATUS_BAD_SLOT
    k, v = b.k64[0], b.v64[0]
    seen = np.r_[0:at * P, (at + 1) * P:n]
    b.k64[0], b.v64[0], b.lens = k[seen], v[seen], [len(seen)]
    b.check(got)
    b.k64[0], b.v64[0], b.lens, b.table = k, v, [n], keep
    kk, vv = torch.randn(1, heads, D, device=DEV), torch.randn(1, heads, D, device=DEV)
    kk[0, 0, 3], vv[0, heads - 1, 40] = float("inf"), float("nan")
    ops.kv_q4_store(b.cache, kk, vv, dev(b.slots(0, np.array([n - 1]))))
    got = b.run()
    b.check(got, but=[(new - 1, slice(None))])
    R = Hq // heads
    assert torch.isnan(got[new - 1, :R]).all()
    if heads > 1:
        last = got[new - 1, -R:]
        assert torch.isnan(last[:, 32:64]).all() and torch.isfinite(last[:, :32]).all() and torch.isfinite(last[:, 64:]).all()
    assert status() == 0


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_many_rows_whatever_the_workspace_holds(typ):
    b = Batch(62, 1, 128, 64, [2600, 300, 40], [140, 1, 2], typ, 8)
    try:
        for size in (40 << 10, 3 << 20, 9 << 20):
            torch.cuda.synchronize()
            ops.shutdown()
            ops.init(0, size)
            b.check(b.run())
    finally:
        torch.cuda.synchronize()
        ops.shutdown()
        ops.init(0, 512 << 20)


@pytest.mark.parametrize("Hq,heads", [(1, 1), (64, 1), (96, 1), (200, 1), (24, 8)])
@pytest.mark.parametrize("typ", ["f32", "f16"])
@pytest.mark.parametrize("lens,new", [([200], [1]), ([200, 90], [1, 2]), ([300], [9])])
def test_groups_of_every_size(Hq, heads, typ, lens, new):
    """One query head per kv head, groups that fill several tiles, and ones past a small request's most rows."""
    b = Batch(Hq, heads, 64, 64, lens, new, typ, Hq)
    b.check(b.run())
    assert status() == 0


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("new", [[1, 2], [140, 1]])
@pytest.mark.parametrize("qmul,kmul,scale", [(1e-4, 1e-3, 2.0**20), (1e-3, 1e3, 1.0), (1e3, 1e-3, 1.0), (1e3, 1e3, 2.0**-20)])
def test_scales_and_magnitudes(typ, new, qmul, kmul, scale):
    """kq_scale at both ends of its range, small and large rows, keys behind a row masked all the same."""
    lens = [200, 40]
    b = Batch(63, 1, 128, 64, lens, new, typ, 8, qstd=2.0 * qmul, kmul=lambda i, n: np.full(n, kmul))
    b.check(b.run(scale=scale), scale=scale)


@pytest.mark.parametrize("new", [1, 140])
def test_zero_and_tiny_rows_average_what_they_see(new):
    b = Batch(64, 1, 64, 32, [170], [new], "f32", 8)
    for x in (0.0, 1e-38, 1e-30, -1e-25):
        b.q.fill_(x)
        b.q64 = np.full(b.q64.shape, np.float64(np.float32(x)))
        b.check(b.run(scale=2.0**-20), scale=2.0**-20)
    assert status() == 0


def test_many_requests():
    """The most requests a call takes, some empty, some of many rows."""
    rng = np.random.default_rng(65)
    S = 4096
    lens, new = rng.integers(0, 3, S), np.ones(S, np.int64)
    new[rng.random(S) < 0.3] = 0
    lens = np.maximum(lens, new)
    lens[[5, 2048, 4095]], new[[5, 2048, 4095]] = [90, 150, 40], [80, 70, 33]
    b = Batch(66, 1, 64, 32, [int(x) for x in lens], [int(x) for x in new], "f16", 4)
    b.check(b.run(), requests=[0, 1, 2, 3, 5, 63, 64, 65, 2047, 2048, 2049, 4000, 4093, 4094, 4095])
    assert status() == 0


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_replayed_prefill_beside_other_calls(typ):
    """A captured call of many rows, replayed after the cache and the lengths it reads have changed and between eager
    calls that use the same workspace."""
    b = Batch(67, 1, 128, 64, [1500], [150], typ, 8)
    other = Batch(68, 1, 128, 64, [4000, 2000], [1, 2], typ, 8)
    want_other = other.run()
    out = torch.zeros_like(b.q)
    table, start, lens = dev(b.table), i32(b.start), i32(b.lens)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attn_kv_q4(b.cache, b.q, table, start, lens, 150, 1500, out=out)
    for n in (1500, 700, 1499, 150):
        lens.copy_(i32([n]))
        out.zero_()
        g.replay()
        assert torch.equal(other.run(), want_other)
        k, v = b.k64[0], b.v64[0]
        b.k64[0], b.v64[0], b.lens = k[:n], v[:n], [n]
        torch.cuda.synchronize()
        b.check(out)
        b.k64[0], b.v64[0], b.lens = k, v, [1500]
    assert status() == 0


# ---- requests whose cells are shared out by the lengths at hand --------------------------


@pytest.mark.parametrize("typ,D,heads,Hq", [("f32", 128, 1, 8), ("bf16", 128, 4, 32), ("f16", 64, 2, 14), ("f32", 256, 2, 16)])
@pytest.mark.parametrize("S", [2, 3, 30, 63, 64, 65])
def test_ragged_decode(typ, D, heads, Hq, S):
    """One long request among short ones, idle ones, one of many rows, one without keys, one beyond the bound."""
    rng = np.random.default_rng(S + D)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(900), S)).astype(int)]
    new = [1] * S
    lens[S // 2] = 2777
    if S > 3:
        lens[1], new[2], lens[3], new[4], lens[4] = 0, 0, 3, 5, 700
    if S == 30:
        lens[7], new[7] = 300, 260                      # (many rows)
    b = Batch(70 + S, heads, D, 64, lens, new, typ, Hq, pad=2)
    out = torch.full_like(b.q, 5.0)
    b.run(out=out)
    b.check(out)
    assert status() == 0
    assert torch.equal(out[b.start[-1]:], torch.full_like(out[b.start[-1]:], 5.0))
    first = out.clone()
    b.run(out=out)
    assert torch.equal(out, first)
    got = b.run(max_len=2776, max_new=max(new))         # the long one is beyond the bound
    assert status() == qa.STATUS_BAD_SEQ
    i = int(b.start[S // 2])
    assert torch.count_nonzero(got[i:i + 1]) == 0
    b.check(got, requests=[x for x in range(S) if x != S // 2])


def test_ragged_lengths_change_between_replays():
    """The shares follow the lengths on the device: one captured call over several sets of them."""
    lens, new = [3000, 40, 700, 1, 90, 2000], [1, 2, 1, 1, 3, 1]
    b = Batch(71, 2, 128, 64, lens, new, "f32", 16)
    out = torch.zeros_like(b.q)
    table, start, there = dev(b.table), i32(b.start), i32(lens)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attn_kv_q4(b.cache, b.q, table, start, there, 3, 3000, out=out)
    k, v = b.k64, b.v64
    for now in (lens, [1, 1, 1, 1, 3, 1], [10, 33, 700, 0, 64, 1999], [3000, 40, 1, 1, 5, 2], [0] * 6, lens):
        there.copy_(i32(now))
        out.fill_(9.0)
        g.replay()
        (torch.randn(1000, device=DEV) ** 2).sum().item()
        torch.cuda.synchronize()
        b.k64, b.v64, b.lens = [x[:n] for x, n in zip(k, now)], [x[:n] for x, n in zip(v, now)], now
        b.check(out)
    assert status() == 0


def test_ragged_lengths_in_odd_orders():
    """Rows of seq_start that lie outside the call or fall back leave the other requests as they are."""
    b = Batch(72, 1, 64, 64, [900, 500, 40], [1, 1, 1], "f16", 8)
    want = b.run()
    for start in ([0, 1, 2, 2], [0, 1, 2, 9], [0, 1, 2, 0]):
        out = torch.full_like(b.q, 5.0)
        b.start = np.array(start)
        b.run(out=out)
        assert torch.equal(out[2], torch.full_like(out[2], 5.0))
        for i in (0, 1):
            w, o = want[i].double(), out[i].double()
            assert float((w - o).abs().max()) <= 2.0**-8 * float(w.abs().max())   # (shares, so sums' orders, differ)


@pytest.mark.parametrize("typ", list(TYPES))
@pytest.mark.parametrize("D,heads,Hq", [(128, 1, 8), (64, 2, 4), (256, 1, 3)])
@pytest.mark.parametrize("lens,new,max_new", [([90, 300, 200], [1, 140, 2], 2), ([300, 90], [200, 1], 1), ([300], [260], 1),
                                              ([400, 300, 90], [300, 150, 1], 150), ([90, 40], [2, 3], 0), ([300], [150], 0)])
def test_many_rows_beyond_max_new(typ, D, heads, Hq, lens, new, max_new):
    """A request of more rows than the bound names gets zeros and a status, however many they are; the others their result."""
    b = Batch(80, heads, D, 64, lens, new, typ, Hq, pad=2)
    out = torch.full_like(b.q, 5.0)
    b.run(out=out, max_new=max_new)
    assert status() == qa.STATUS_BAD_SEQ
    for i, n in enumerate(new):
        if n > max_new:
            assert torch.count_nonzero(out[b.start[i]:b.start[i + 1]]) == 0
    b.check(out, requests=[i for i, n in enumerate(new) if n <= max_new])
    assert torch.equal(out[b.start[-1]:], torch.full_like(out[b.start[-1]:], 5.0))


@pytest.mark.parametrize("new", [[1], [1, 3], [150, 1]])
def test_no_keys_at_all(new):
    b = Batch(81, 1, 128, 32, [0] * len(new), new, "bf16", 8)
    out = torch.full_like(b.q, 5.0)
    b.run(out=out, max_len=0)
    assert torch.count_nonzero(out) == 0 and status() == 0


def test_requests_that_share_pages():
    """Two requests over one prefix's pages, and a page that occurs twice in a request."""
    b = Batch(82, 2, 128, 64, [192, 200, 192], [1, 4, 130], "f32", 8)
    b.table[1, :2] = b.table[0, :2]
    b.table[2, 2] = b.table[2, 0]
    for x in (b.k64, b.v64):
        x[1][:128] = x[0][:128]
        x[2][128:] = x[2][:64]
    b.check(b.run())
    assert status() == 0
