"""ix_rope_rows against tests/rope_ref.py in 64 bits: within half a bf16 step (2^-8) of the result and what its 32-bit
arithmetic may be off by (derived there). ix_kv8_append_rope: its queries are ix_rope_rows' and its cache is that of
ix_kv8_append on ix_rope_rows' keys, bit for bit."""
import ctypes
import math

import numpy as np
import pytest

import baloon_amd as bx
from tests import kv8_ref, rope_ref
from tests.test_kv8_cache import Pair, bf, cumulative, desc, ints, tables_for

INVALID = bx.HIP_ERROR_INVALID_VALUE
A = 1 << 20


def description(rot=64, layout=0, freq=A, amplitude=1.0, norm=None, offset=0.0, eps=1e-6):
    return bx.Rope(rot, layout, freq, amplitude, norm, offset, eps)


def rows_of(x):
    return None if x is None else ctypes.byref(bx.Rows(*x))


def rope(r=None, n_seq=2, T=4, cu=A, kv=A, x=(A, 256), heads=4, d=64, y=A):
    return bx.lib().ix_rope_rows(None if r == 0 else ctypes.byref(r or description()), n_seq, T, cu, kv, rows_of(x), heads, d, y, None)


def append(c=None, n_seq=2, T=4, cu=A, kv=A, table=A, width=3, k=(A, 128), v=(A, 128), rk=None, q=(A, 256), h_q=4, rq=None, out=A):
    rk, rq = (None if r == 0 else ctypes.byref(r or description()) for r in (rk, rq))
    return bx.lib().ix_kv8_append_rope(ctypes.byref(c or desc()), n_seq, T, cu, kv, table, width, rows_of(k), rows_of(v), rk, rows_of(q),
                                       h_q, rq, out, None)


BAD = [dict(rot=-2), dict(rot=63), dict(rot=66), dict(layout=2), dict(layout=-1), dict(freq=None), dict(freq=A + 2), dict(norm=A + 1)]


def test_refusals():
    for kw in BAD:
        assert rope(description(**kw)) == INVALID, kw
        assert append(rk=description(**kw)) == INVALID and append(rq=description(**kw)) == INVALID, kw
    assert rope(0) == INVALID and append(rk=0) == INVALID and append(rq=0) == INVALID
    for kw in (dict(n_seq=0), dict(n_seq=65536), dict(T=-1), dict(cu=None), dict(kv=None), dict(cu=A + 2), dict(kv=A + 1)):
        assert rope(**kw) == INVALID and append(**kw) == INVALID, kw
    for kw in (dict(x=None), dict(x=(None, 256)), dict(x=(A + 1, 256)), dict(x=(A, 255)), dict(x=(A, -256)), dict(heads=0), dict(heads=-1),
               dict(heads=65537, x=(A, 1 << 40)), dict(d=60), dict(d=0), dict(d=-64), dict(d=520, x=(A, 4096)), dict(d=56), dict(y=None), dict(y=A + 1)):
        assert rope(**kw) == INVALID, kw
    for kw in (dict(k=None), dict(k=(A, 127)), dict(v=None), dict(v=(A + 1, 128)), dict(q=(None, 256)), dict(q=(A, 255)), dict(h_q=0),
               dict(h_q=65537, q=(A, 1 << 40)), dict(out=None), dict(out=A + 1), dict(c=desc(page=48)), dict(c=desc(d=96)), dict(table=None),
               dict(width=0)):
        assert append(**kw) == INVALID, kw


def test_no_rows():
    assert rope(T=0, x=(None, 256), y=None) == bx.HIP_SUCCESS
    assert append(T=0, k=(None, 128), v=(None, 128), q=(None, 256), out=None) == bx.HIP_SUCCESS
    assert append(T=0, q=None, h_q=0, rq=0, out=None) == bx.HIP_SUCCESS
    assert rope(0, T=0) == INVALID and rope(T=0, d=60) == INVALID and append(T=0, rk=0) == INVALID and append(T=0, rq=0) == INVALID


def test_mirror_refusals():
    import torch
    with pytest.raises(ValueError, match="fp32"):
        bx.rope(torch.zeros(8, dtype=torch.float64))
    with pytest.raises(ValueError, match="one dimension"):
        bx.rope(torch.zeros(8, 2))
    with pytest.raises(ValueError, match="on the GPU"):
        bx.rope(torch.zeros(8))
    with pytest.raises(TypeError):
        bx.ix_rope_rows(ctypes.c_int(1), 1, 1, None, None, None, 1, 64, None, 0)
    assert bx.ix_rope_rows(None, 1, 1, None, None, None, 1, 64, None, 0) == INVALID
    short = description()
    short.tensors = (None, torch.ones(32))
    for call in (lambda: bx.ix_rope_rows(short, 1, 1, None, None, None, 1, 64, None, 0),
                 lambda: bx.ix_kv8_append_rope(desc(), 1, 1, None, None, None, 1, None, None, short),
                 lambda: bx.ix_kv8_append_rope(desc(), 1, 1, None, None, None, 1, None, None, None, bx.Rows(A, 256), 4, short)):
        with pytest.raises(ValueError, match="weight for each"):
            call()


def test_frequencies():
    plain, one = bx.rope_freq(64, 1e4)
    i = np.arange(32)
    assert one == 1.0 and np.allclose(plain, 1e4 ** (-i / 32), rtol=2.0 ** -23)
    assert np.allclose(bx.rope_freq(64, 1e4, "linear", 8.0)[0], plain / 8, rtol=2.0 ** -22)
    base, one = bx.rope_freq(64, 1e4, "base", 8.0)
    assert one == 1.0 and base[0] == plain[0] and math.isclose(base[-1], plain[-1] / 8, rel_tol=2.0 ** -22)
    parts, more = bx.rope_freq(64, 1e4, "parts", 4.0, trained=4096)
    rounds = 4096 * 1e4 ** (-i / 32) / (2 * np.pi)
    assert math.isclose(more, 0.1 * math.log(4) + 1)
    assert np.allclose(parts[rounds > 32], plain[rounds > 32], rtol=2.0 ** -22)
    assert np.allclose(parts[rounds < 1], plain[rounds < 1] / 4, rtol=2.0 ** -22)
    between = (rounds > 1) & (rounds < 32)
    assert between.any() and np.all((parts < plain).numpy()[between] & (parts > plain / 4).numpy()[between])
    assert np.allclose(bx.rope_freq(2, 1e4, "base", 8.0)[0], [1.0])
    for args in ((63,), (0,), (64, 0.5), (64, 1e4, "linear", 0.5), (64, 1e4, "parts", 2.0), (64, 1e4, "other")):
        with pytest.raises(ValueError):
            bx.rope_freq(*args)


# ---- on the GPU --------------------------------------------------------------------------------

def make(g, d, rot, layout=bx.ROPE_HALVES, norm=True, amplitude=1.0, base=1e4, offset=1.0, eps=1e-6):
    """(description, the same as rope_ref.turned takes it)"""
    import torch
    freq = (base ** (-np.arange(rot // 2) / max(rot // 2, 1))).astype(np.float32)
    w = (g.standard_normal(d) * 0.3).astype(np.float32) if norm else None
    r = bx.rope(torch.from_numpy(freq).cuda() if rot else None, layout, amplitude, None if w is None else torch.from_numpy(w).cuda(), offset, eps)
    return r, dict(freq=freq, pairs=layout == bx.ROPE_PAIRS, amplitude=np.float32(amplitude), norm=w, offset=offset, eps=eps)


def positions(q, kv):
    return np.concatenate([np.arange(n - m, n) for m, n in zip(q, kv)]) if sum(q) else np.zeros(0)


def near(got, x, pos, ref):
    want, off = rope_ref.turned(x, pos, **ref)
    bad = np.abs(got - want) > 2.0 ** -8 * np.abs(want) + 2.0 ** -8 * off + off
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


ROWS = [  # d, heads, rot, layout, norm, amplitude
    (64, 1, 64, 0, False, 1.0), (64, 3, 32, 1, True, 1.0), (64, 17, 2, 0, True, 1.25), (64, 2, 2, 1, False, 1.0), (64, 5, 0, 0, True, 1.0),
    (80, 4, 80, 0, True, 1.0), (80, 33, 32, 1, False, 1.0), (96, 2, 24, 0, True, 1.0), (8, 9, 8, 0, True, 1.0), (16, 5, 6, 1, True, 1.0),
    (128, 32, 128, 1, False, 1.0), (128, 8, 128, 0, True, 0.7), (128, 4, 126, 0, True, 1.0), (128, 4, 126, 1, True, 1.0),
    (192, 3, 64, 0, False, 1.0), (256, 16, 64, 0, True, 1.0), (256, 2, 256, 0, False, 1.0), (256, 7, 20, 0, True, 1.0),
    (256, 9, 250, 1, True, 1.0), (264, 2, 200, 0, True, 1.0), (512, 3, 512, 0, True, 1.0), (512, 2, 34, 1, False, 1.0), (72, 2, 0, 1, False, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,rot,layout,norm,amplitude", ROWS)
@pytest.mark.parametrize("how", ["packed", "slice", "odd", "in place"])
def test_rows(d, heads, rot, layout, norm, amplitude, how):
    import torch
    g = np.random.default_rng(d + heads + rot)
    q, kv = [1, 0, 37, 5], [1001, 9, 40, 5]
    T = sum(q)
    bits, x = kv8_ref.normal_bf16(g, T, heads, d)
    if how == "slice":
        wide = torch.zeros(T, heads + 2, d, dtype=torch.bfloat16, device="cuda")
        wide[:, :heads] = bf(bits)
        rows = wide[:, :heads]
    elif how == "odd":
        wide = torch.zeros(T, heads * d + 1, dtype=torch.bfloat16, device="cuda")
        wide[:, 1:] = bf(bits).view(T, -1)
        rows = wide[:, 1:]
    else:
        rows = bf(bits)
    r, ref = make(g, d, rot, layout, norm, amplitude)
    y = rows if how == "in place" else torch.full((T, heads, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    assert bx.ix_rope_rows(r, len(q), T, ints(cumulative(q)), ints(kv), rows, heads, d, y) == 0
    near(y.float().cpu().numpy(), x, positions(q, kv), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("base", [1e4, 1e7])
def test_far(layout, base):
    """Positions up to 2^30, where an angle in 32 bits would be off by whole turns; and before 0."""
    import torch
    g = np.random.default_rng(3)
    q, kv = [3, 2, 4, 2], [1 << 30, 999999, 2, (1 << 24) + 1]
    bits, x = kv8_ref.normal_bf16(g, 11, 4, 128)
    r, ref = make(g, 128, 128, layout, False, base=base)
    y = torch.empty(11, 4, 128, dtype=torch.bfloat16, device="cuda")
    assert bx.ix_rope_rows(r, 4, 11, ints(cumulative(q)), ints(kv), bf(bits), 4, 128, y) == 0
    near(y.float().cpu().numpy(), x, positions(q, kv), ref)


@pytest.mark.gpu
def test_many_sequences_and_rows_of_none():
    """5,000 sequences, many of them empty, whose offsets begin behind the first row and end before the last."""
    import torch
    g = np.random.default_rng(4)
    q = g.integers(0, 3, 5000)
    kv = q + g.integers(0, 5000, 5000)
    n, before, behind = int(q.sum()), 5, 7
    T = before + n + behind
    bits, x = kv8_ref.normal_bf16(g, T, 2, 64)
    r, ref = make(g, 64, 32)
    y = torch.full((T, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    assert bx.ix_rope_rows(r, 5000, T, ints(before + np.array(cumulative(q))), ints(kv), bf(bits), 2, 64, y) == 0
    got = y.float().cpu().numpy()
    assert np.all(got[:before] == 7) and np.all(got[before + n:] == 7)
    near(got[before:before + n], x[before:before + n], positions(q, kv), ref)


@pytest.mark.gpu
def test_values_that_are_none():
    """An infinite or NaN channel stays in its pair, and one that passes passes."""
    import torch
    x = torch.ones(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    x[0, 0, 5], x[0, 0, 34], x[0, 0, 35] = float("nan"), float("inf"), float("-inf")
    for layout in (0, 1):
        r, _ = make(np.random.default_rng(0), 64, 34, layout, False)
        y = torch.empty_like(x)
        assert bx.ix_rope_rows(r, 1, 1, ints([0, 1]), ints([8]), x, 1, 64, y) == 0
        y = y[0, 0]
        mate = 22 if layout == 0 else 4
        others = torch.tensor([c for c in range(64) if c not in (5, mate, 34, 35)], device="cuda")
        assert bool(y[[5, mate]].isnan().all()) and bool(y[others].isfinite().all())
        assert y[34] == float("inf") and y[35] == float("-inf")


@pytest.mark.gpu
def test_eps_and_rows_of_zeros():
    import torch
    g = np.random.default_rng(5)
    for eps in (1e-6, 1e-2):
        bits, x = kv8_ref.normal_bf16(g, 4, 2, 128, std=1e-3)
        bits[1], x[1] = 0, 0
        r, ref = make(g, 128, 64, eps=eps, offset=0.0)
        y = torch.empty(4, 2, 128, dtype=torch.bfloat16, device="cuda")
        assert bx.ix_rope_rows(r, 1, 4, ints([0, 4]), ints([4]), bf(bits), 2, 128, y) == 0
        near(y.float().cpu().numpy(), x, np.arange(4), ref)


APPEND = [  # page, h_kv, d, G, rot, layout, norm
    (16, 2, 64, 2, 64, 0, True), (32, 1, 64, 1, 16, 1, False), (64, 3, 128, 4, 128, 0, False), (128, 1, 128, 8, 64, 1, True),
    (16, 2, 256, 8, 64, 0, True), (64, 1, 256, 3, 256, 1, True), (128, 1, 256, 1, 256, 0, True), (32, 2, 128, 2, 20, 0, True),
    (16, 1, 128, 2, 126, 1, False), (64, 2, 64, 5, 0, 0, True), (128, 2, 64, 16, 62, 0, False),
]


def append_both(p, q, lens, tables, h_q, rk, rq, how="slice"):
    """One append through the library; the reference's on keys that ix_rope_rows has turned."""
    import torch
    h, d = p.ref.h, p.ref.d
    T, cu = sum(q), cumulative(q)
    bits, x = kv8_ref.normal_bf16(p.g, T, h_q + 2 * h, d)
    if how == "odd":
        wide = torch.zeros(T, (h_q + 2 * h) * d + 1, dtype=torch.bfloat16, device="cuda")
        wide[:, 1:] = bf(bits).view(T, -1)
        rows = wide[:, 1:]
    else:
        rows = bf(bits).view(T, -1)
    qs, k, v = rows.split([h_q * d, h * d, h * d], 1)
    batch = (len(q), T, ints(cu), ints(lens))
    want_q, want_k = (torch.empty(T, n, d, dtype=torch.bfloat16, device="cuda") for n in (h_q, h))
    assert bx.ix_rope_rows(rq, *batch, qs, h_q, d, want_q) == 0 and bx.ix_rope_rows(rk, *batch, k, h, d, want_k) == 0
    out = torch.full_like(want_q, float("nan"))
    assert bx.ix_kv8_append_rope(p.cache, *batch, ints(tables), tables.shape[1], k, v, rk, qs, h_q, rq, out) == 0
    assert torch.equal(out.view(torch.int16), want_q.view(torch.int16))
    turned = want_k.float().cpu().numpy()
    for b, m in enumerate(q):
        s = slice(cu[b], cu[b + 1])
        p.ref.append(m, lens[b], tables[b], {"k": turned[s], "v": x[s, h_q + h:]})
    p.check(lens, tables)


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d,G,rot,layout,norm", APPEND)
@pytest.mark.parametrize("how", ["slice", "odd"])
def test_append(page, h, d, G, rot, layout, norm, how):
    """Prompts, single tokens and drafts onto pages that are fresh, half filled and full; an empty sequence among them."""
    p = Pair(40, page, h, d, page + d + rot)
    lens = [0, 0, 0]
    todo = [(3 * page + 5, 0, 1), (1, 1, 1), (2, page - 2, 0), (4, 4, 4), (1, 1, 1)]
    most = [sum(t[b] for t in todo) for b in range(3)]
    tables = tables_for(p.g, 40, most, page, max(-(-n // page) for n in most) + 1)
    (rk, _), (rq, _) = make(p.g, d, rot, layout, norm), make(p.g, d, min(d, rot + 16) if rot else d, 1 - layout, not norm)
    for q in todo:
        lens = [n + m for n, m in zip(lens, q)]
        append_both(p, list(q), lens, tables, G * h, rk, rq, how)


@pytest.mark.gpu
def test_append_of_many_queries():
    """More than 2^24 values of queries."""
    p = Pair(72, 64, 1, 256, 12)
    tables = tables_for(p.g, 72, [4140, 35], 64, 66)
    (rk, _), (rq, _) = make(p.g, 256, 64), make(p.g, 256, 256, 1, False)
    append_both(p, [4100, 5], [4100, 5], tables, 16, rk, rq)
    append_both(p, [1, 30], [4101, 35], tables, 16, rk, rq)


@pytest.mark.gpu
def test_append_places():
    """Pages without a place, tokens before position 0, offsets behind the first row; no queries, and queries in place."""
    import torch
    p = Pair(12, 16, 2, 64, 9)
    tables = np.array([[3, -1, 5, 99], [7, 0, 1, 2]], np.int32)
    rk, _ = make(p.g, 64, 32)
    rq, _ = make(p.g, 64, 64, 1, False)
    append_both(p, [50, 20], [50, 12], tables, 4, rk, rq)
    bits, x = kv8_ref.normal_bf16(p.g, 9 + 3, 4, 64)
    rows = bf(bits)
    q, k, v = rows[:, :2].contiguous(), rows[:, 2:3].contiguous().expand(-1, 2, -1).contiguous(), rows[:, 2:]
    cu, kv = ints([9, 10, 12]), ints([51, 14])
    want_k, want_q = torch.empty_like(k), q.clone()
    assert bx.ix_rope_rows(rk, 2, 12, cu, kv, k, 2, 64, want_k) == 0 and bx.ix_rope_rows(rq, 2, 12, cu, kv, q, 2, 64, want_q) == 0
    for queries in (False, True):
        more = (q, 2, rq, q) if queries else ()
        assert bx.ix_kv8_append_rope(p.cache, 2, 12, cu, kv, ints(tables), 4, k, v, rk, *more) == 0
        for b, s in enumerate((slice(9, 10), slice(10, 12))):
            p.ref.append(s.stop - s.start, (51, 14)[b], tables[b], {"k": want_k.float().cpu().numpy()[s], "v": x[s, 2:]})
        p.check([51, 14], tables)
    assert torch.equal(q, want_q) and torch.equal(q[:9], bf(bits)[:9, :2])


@pytest.mark.gpu
def test_captured():
    """A graph of the append on another stream than torch's current one, replayed with other lengths and rows."""
    import torch
    g = np.random.default_rng(11)
    cache, again = ([torch.zeros(s, dtype=t, device="cuda") for s, t in (((8, 2, 16, 64), torch.int8), ((8, 2, 64, 16), torch.int8),
                                                                         ((8, 2), torch.float32), ((8, 2), torch.float32))] for _ in "ab")
    c1, c2 = bx.kv8_cache(*cache), bx.kv8_cache(*again)
    rk, _ = make(g, 64, 32)
    rows = torch.empty(3, 8, 64, dtype=torch.bfloat16, device="cuda")
    kv, cu, table = ints([1, 1, 1]), ints([0, 1, 2, 3]), ints([[0, 1], [2, 3], [4, 5]])
    out, want = torch.empty(3, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(3, 4, 64, dtype=torch.bfloat16, device="cuda")

    def call(c, o, s=None):
        assert bx.ix_kv8_append_rope(c, 3, 3, cu, kv, table, 2, rows[:, 4:6], rows[:, 6:], rk, rows[:, :4], 4, rk, o, s) == 0

    stream = torch.cuda.Stream()
    rows.normal_()
    call(c2, want, stream)
    torch.cuda.synchronize()
    for t in again:
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(c1, out)
    for i in range(20):
        rows.normal_()
        kv.fill_(i + 1)
        torch.cuda.synchronize()
        graph.replay()
        call(c2, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(cache, again)), i
