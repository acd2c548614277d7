"""ix_kv8_append and ix_kv8_read. The cache's codes and scales are defined in IEEE fp32, so they are compared with
tests/kv8_ref.py bit for bit, at every position the sequences hold; what ix_kv8_read gives is the bf16 rounding of
scale * code, bit for bit."""
import ctypes

import numpy as np
import pytest

import baloon_amd as bx
from oracle import bf16
from tests import kv8_ref

INVALID = bx.HIP_ERROR_INVALID_VALUE
A = 1 << 20


def desc(n_pages=8, page=16, h=2, d=64, k=A, v=A, ks=A, vs=A):
    return bx.Kv8(n_pages, page, h, d, k, v, ks, vs)


def append(c=None, n_seq=2, T=4, cu=A, kv=A, table=A, width=3, k=(A, 128), v=(A, 128)):
    r = [None if x is None else ctypes.byref(bx.Rows(*x)) for x in (k, v)]
    return bx.lib().ix_kv8_append(ctypes.byref(c or desc()), n_seq, T, cu, kv, table, width, *r, None)


def read(c=None, n_seq=2, T=4, cu=A, kv=A, table=A, width=3, k=A, v=A):
    return bx.lib().ix_kv8_read(ctypes.byref(c or desc()), n_seq, T, cu, kv, table, width, k, v, None)


def test_refusals():
    bad = [desc(n_pages=0), desc(page=8), desc(page=24), desc(page=256), desc(h=0), desc(h=1025), desc(d=32), desc(d=96),
           desc(d=512), desc(k=None), desc(v=None), desc(ks=None), desc(vs=None), desc(k=A + 8), desc(v=A + 8), desc(ks=A + 2),
           desc(vs=A + 2)]
    for f in (append, read):
        for c in bad:
            assert f(c) == INVALID, [getattr(c, n) for n, _ in c._fields_]
        for kw in (dict(n_seq=0), dict(n_seq=-1), dict(n_seq=65536), dict(T=-1), dict(cu=None), dict(kv=None), dict(table=None),
                   dict(width=0), dict(cu=A + 2), dict(kv=A + 1), dict(table=A + 2)):
            assert f(**kw) == INVALID, kw
        assert f(T=0) == bx.HIP_SUCCESS
    assert bx.lib().ix_kv8_append(None, 2, 4, A, A, A, 3, ctypes.byref(bx.Rows(A, 128)), ctypes.byref(bx.Rows(A, 128)), None) == INVALID
    for r in (None, (None, 128), (A, 127), (A, -128), (A + 1, 128)):
        assert append(k=r) == INVALID and append(v=r) == INVALID, r
    assert read(k=None, v=None) == INVALID
    assert read(k=A + 1) == INVALID and read(v=A + 1) == INVALID


def test_mirror_refusals():
    import torch
    t = torch.zeros
    with pytest.raises(ValueError, match="must be on the GPU"):
        bx.ix_kv8_append(desc(), 1, 1, None, None, None, 1, t(1, 128, dtype=torch.bfloat16), None, 0)
    with pytest.raises(TypeError):
        bx.ix_kv8_append(ctypes.c_int(1), 1, 1, None, None, None, 1, None, None, 0)
    with pytest.raises(ValueError, match="n_pages"):
        bx.kv8_cache(t(4, 2, 16, 64, dtype=torch.int8), t(4, 2, 16, 64, dtype=torch.int8), t(4, 2), t(4, 2))
    with pytest.raises(ValueError, match="scales"):
        bx.kv8_cache(t(4, 2, 16, 64, dtype=torch.int8), t(4, 2, 64, 16, dtype=torch.int8), t(4), t(4, 2))
    with pytest.raises(ValueError, match="int8"):
        bx.kv8_cache(t(4, 2, 16, 64), t(4, 2, 64, 16), t(4, 2), t(4, 2))
    assert bx.ix_kv8_append(None, 1, 1, None, None, None, 1, None, None, 0) == INVALID
    assert bx.ix_kv8_append(desc(), 1, 1, None, None, None, 1, bx.Rows(A, 3), bx.Rows(A, 128), 0) == INVALID


# ---- on the GPU --------------------------------------------------------------------------------

class Pair:
    """The library's cache and the reference's, of the same content."""

    def __init__(self, n_pages, page, h, d, seed):
        import torch
        self.g = np.random.default_rng(seed)
        self.ref = kv8_ref.Cache(n_pages, page, h, d, self.g)
        c, s = self.ref.codes, self.ref.scale
        self.t = [torch.from_numpy(x).cuda() for x in (c["k"].copy(), np.ascontiguousarray(c["v"].swapaxes(2, 3)), s["k"].copy(),
                                                        s["v"].copy())]
        self.cache = bx.kv8_cache(*self.t)

    def check(self, kv_len, tables):
        """Every code that a sequence holds, and every scale, bit for bit."""
        k, v, ks, vs = (t.cpu().numpy() for t in self.t)
        v = v.swapaxes(2, 3)
        assert np.array_equal(ks.view(np.int32), self.ref.scale["k"].view(np.int32))
        assert np.array_equal(vs.view(np.int32), self.ref.scale["v"].view(np.int32))
        for n, table in zip(kv_len, tables):
            for p in range(-(-n // self.ref.page)):
                at = self.ref.place(table, p)
                if at is not None:
                    m = min(self.ref.page, n - p * self.ref.page)
                    assert np.array_equal(k[at, :, :m], self.ref.codes["k"][at, :, :m]), (p, at)
                    assert np.array_equal(v[at, :, :m], self.ref.codes["v"][at, :, :m]), (p, at)


def ints(v):
    import torch
    return torch.tensor(np.asarray(v), dtype=torch.int32).cuda()


def bf(bits):
    import torch
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16).copy()).view(torch.bfloat16).cuda()


def cumulative(q):
    return [0] + list(np.cumsum(q))


def steps(p, q_steps, tables, lens, how="slice", scale=None):
    """Append q_steps[i][b] tokens to sequence b, step by step, and compare everything after each."""
    import torch
    h, d = p.ref.h, p.ref.d
    table = ints(tables)
    for i, q in enumerate(q_steps):
        T, cu = sum(q), cumulative(q)
        lens = [n + m for n, m in zip(lens, q)]
        std = np.float32(1.0 if scale is None else scale[i])
        bits, x = kv8_ref.normal_bf16(p.g, T, 2, h, d, std=std)
        if how == "slice":                                     # of wider rows, as a projection leaves them
            rows = torch.zeros(T, 3, h, d, dtype=torch.bfloat16, device="cuda")
            rows[:, :2] = bf(bits)
            k, v = rows[:, 0], rows[:, 1]
        elif how == "odd":                                     # rows of an odd stride
            rows = torch.zeros(T, 2 * h * d + 1, dtype=torch.bfloat16, device="cuda")
            rows[:, :-1] = bf(bits).view(T, -1)
            k, v = rows[:, :h * d], rows[:, h * d:-1]
        else:
            k, v = bf(bits[:, 0]), bf(bits[:, 1])
        args = (p.cache, len(q), T, ints(cu), ints(lens), table, table.shape[1])
        assert bx.ix_kv8_append(*args, k, v) == 0
        for b, m in enumerate(q):
            s = slice(cu[b], cu[b + 1])
            p.ref.append(m, lens[b], tables[b], {"k": x[s, 0], "v": x[s, 1]})
        p.check(lens, tables)
        # the new tokens' values, and nothing besides
        out = [torch.full((T, h, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
        assert bx.ix_kv8_read(*args, *out) == 0
        for n, o in zip("kv", out):
            got = o.float().cpu().numpy()
            for b, m in enumerate(q):
                val, has = p.ref.tokens(n, max(lens[b], 0), tables[b])
                at = np.arange(lens[b] - m, lens[b])
                ok = np.array([t >= 0 and has[t] for t in at], bool)
                want = np.full((m, h, d), 7.0, np.float32)
                if m:
                    want[ok] = bf16.to_f32(bf16.from_f32(val[at[ok]]))
                assert np.array_equal(got[cu[b]:cu[b + 1]], want), (n, b)
    return lens


def tables_for(g, n_pages, lens, page, width):
    order = list(g.permutation(n_pages))
    t = np.full((len(lens), width), -1, np.int32)
    for b, n in enumerate(lens):
        for p in range(-(-n // page)):
            t[b, p] = order.pop()
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d", [(16, 2, 256), (16, 3, 64), (32, 1, 128), (64, 2, 128), (64, 1, 64), (128, 1, 256),
                                      (128, 2, 64), (32, 2, 256)])
@pytest.mark.parametrize("how", ["slice", "odd", "packed"])
def test_prompt_then_tokens(page, h, d, how):
    """Prompts of all lengths, then tokens one and some at a time, in pages whose scale grows or stays."""
    p = Pair(64, page, h, d, page * d + h)
    q = [[page + 3, 1, 0, 2 * page, page - 1], [1, 1, 1, 1, 1], [1, 0, 1, 0, 1], [5, 17, page, 2, 1], [1, 1, 1, 1, 1]]
    ends = list(np.sum(q, 0))
    tables = tables_for(p.g, 64, ends, page, -(-max(ends) // page) + 2)
    steps(p, q, tables, [0] * 5, how, scale=[1.0, 0.5, 3.0, 1.0, 20.0])


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq", [1, 63, 64, 65, 130, 4100])
def test_many_sequences(n_seq):
    """The search for a page's sequence at one, two and three steps, with sequences that have nothing new."""
    g = np.random.default_rng(n_seq)
    p = Pair(2 * n_seq + 40, 16, 1, 64, n_seq)
    q = [int(x) for x in g.integers(0, 3, n_seq)]
    q[-1] = 20
    q2 = [int(x) for x in g.integers(0, 2, n_seq)]
    tables = tables_for(p.g, p.ref.n_pages, [a + b for a, b in zip(q, q2)], 16, 3)
    steps(p, [q, q2], tables, [0] * n_seq, "packed")


@pytest.mark.gpu
def test_values_at_the_edges():
    """Zeros, the smallest and largest numbers, ties, and a page whose first tokens are all zero."""
    import torch
    p = Pair(4, 16, 1, 64, 3)
    tables = np.array([[2]], np.int32)
    lens = 0
    for x in (np.zeros(64), np.full(64, 1e-40), np.full(64, 1e-38), np.linspace(-127, 127, 64), np.arange(64) + 0.5,
              np.full(64, 3e38), np.full(64, -3e38), np.zeros(64)):
        bits = bf16.from_f32(np.stack([x, -x]).astype(np.float32).reshape(2, 1, 64))
        val = bf16.to_f32(bits)
        lens += 2
        k, v = bf(bits), bf(bits[::-1].copy())
        assert bx.ix_kv8_append(p.cache, 1, 2, ints([0, 2]), ints([lens]), ints(tables), 1, k, v) == 0
        p.ref.append(2, lens, tables[0], {"k": val, "v": val[::-1]})
        p.check([lens], tables)
    assert np.all(np.isfinite(p.t[2].cpu().numpy()[2]))


@pytest.mark.gpu
def test_pages_without_a_place():
    """Entries outside the cache, positions behind the table and before the sequence's start: dropped."""
    p = Pair(6, 16, 2, 64, 5)
    before = [t.clone() for t in p.t]
    tables = np.array([[1, -1, 2], [6, 3, 1 << 30], [4, 5, -7]], np.int32)
    # the third sequence has fewer tokens than are new; the first is longer than its table
    steps(p, [[40, 40, 20], [30, 5, 3]], tables, [0, 0, -4], "slice")
    import torch
    for page in (0,):                                           # a page of no sequence is as it was
        for a, b in zip(before, p.t):
            assert torch.equal(a[page].nan_to_num(7.0) if a.is_floating_point() else a[page],
                               b[page].nan_to_num(7.0) if b.is_floating_point() else b[page])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    import torch
    n_pages, page, h, d = 700_000, 16, 2, 256                    # 5.7 GB of codes each
    k = torch.empty(n_pages, h, page, d, dtype=torch.int8, device="cuda")
    v = torch.empty(n_pages, h, d, page, dtype=torch.int8, device="cuda")
    s = [torch.empty(n_pages, h, device="cuda") for _ in "kv"]
    cache = bx.kv8_cache(k, v, *s)
    table = [[699_999, 5, 620_000]]
    g = np.random.default_rng(8)
    bits, x = kv8_ref.normal_bf16(g, 40, 2, h, d)
    rows = bf(bits)
    args = (cache, 1, 40, ints([0, 40]), ints([40]), ints(table), 3)
    assert bx.ix_kv8_append(*args, rows[:, 0], rows[:, 1]) == 0
    out = [torch.empty(40, h, d, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    assert bx.ix_kv8_read(*args, *out) == 0
    ref = kv8_ref.Cache(3, page, h, d, g)
    ref.append(40, 40, [0, 1, 2], {"k": x[:, 0], "v": x[:, 1]})
    for i, n in enumerate("kv"):
        assert np.array_equal(out[i].float().cpu().numpy(), bf16.to_f32(bf16.from_f32(ref.tokens(n, 40, [0, 1, 2])[0])))
    # half a quantum of the page's largest value, and bf16's own half ulp
    assert np.all(np.abs(out[0].float().cpu().numpy() - x[:, 0]) <= np.abs(x[:, 0]).max() * (0.5 / 127 + 2.0 ** -8))


@pytest.mark.gpu
def test_row_operands():
    """What the mirror takes as rows, and what it refuses."""
    import torch
    p = Pair(4, 16, 2, 64, 11)
    args = (p.cache, 1, 2, ints([0, 2]), ints([2]), ints([[0]]), 1)
    rows = torch.randn(2, 2, 64, device="cuda").bfloat16()
    assert bx.ix_kv8_append(*args, rows, rows.view(2, 128)) == 0
    assert bx.ix_kv8_append(*args, bx.Rows(rows.data_ptr(), 128), rows) == 0
    assert torch.equal(p.t[0][0, :, :2], p.t[1][0, :, :, :2].transpose(1, 2))     # keys and values were the same
    for bad in (rows.float(), rows.transpose(1, 2), rows[:, :, :32], rows.view(-1)):
        with pytest.raises(ValueError):
            bx.ix_kv8_append(*args, bad, rows)
    assert bx.ix_kv8_append(*args, rows.view(4, 64), rows) == INVALID                 # the tensor's rows are too close
