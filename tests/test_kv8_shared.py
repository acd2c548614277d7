"""ix_kv8_attn_shared against the attention of tests/kv8_ref.py in 64 bits, each sequence over all of its tokens by itself. The
tolerance is that of ix_kv8_attn (tests/test_kv8_attn.py): a row's two partial results are put together in 32 bits, by factors
that are within 2^-22 of theirs, which its (n / 16 + 64) 2^-23 covers."""
import ctypes

import numpy as np
import pytest

import baloon_amd as bx
from tests.test_kv8_attn import Problem
from tests.test_kv8_cache import bf, cumulative, desc, ints

INVALID = bx.HIP_ERROR_INVALID_VALUE
A = 1 << 20


def attn(c=None, n_seq=2, T=4, max_q=2, cu=A, kv=A, table=A, width=3, n_groups=1, groups=A, shared=A, q=(A, 256), h_q=4, gate=None, o=A,
         ws=A, nbytes=1 << 40):
    r = [None if x is None else ctypes.byref(bx.Rows(*x)) for x in (q, gate)]
    return bx.lib().ix_kv8_attn_shared(None if c == 0 else ctypes.byref(c or desc()), n_seq, T, max_q, cu, kv, table, width, n_groups, groups,
                                       shared, r[0], h_q, ctypes.c_float(1), r[1], o, ws, nbytes, None)


def test_refusals():
    assert attn(0) == INVALID
    for c in (desc(n_pages=0), desc(page=48), desc(h=0), desc(d=96), desc(k=None), desc(vs=None), desc(k=A + 4)):
        assert attn(c) == INVALID
    for kw in (dict(n_seq=0), dict(n_seq=65536), dict(T=-1), dict(max_q=0), dict(max_q=-1), dict(cu=None), dict(kv=None), dict(table=None),
               dict(width=0), dict(cu=A + 2), dict(h_q=0), dict(h_q=3), dict(h_q=-4), dict(n_groups=-1), dict(n_groups=65536), dict(groups=None),
               dict(groups=A + 2), dict(shared=None), dict(shared=A + 1), dict(o=None), dict(o=A + 1), dict(ws=None), dict(ws=A + 16),
               dict(q=None), dict(q=(None, 256)), dict(q=(A, 255)), dict(q=(A + 1, 256)), dict(gate=(None, 256)), dict(gate=(A, 255)),
               dict(gate=(A + 1, 256))):
        assert attn(**kw) == INVALID, kw
    need = bx.ix_kv8_attn_shared_workspace_size(desc(), 2, 4, 2, 1, 4)
    assert need >= bx.ix_kv8_attn_workspace_size(desc(), 2, 4, 2, 4) + 4 * 4 * (64 + 2) * 4 and attn(nbytes=need - 1) == INVALID
    assert attn(T=0, max_q=0, q=(None, 256), o=None) == bx.HIP_SUCCESS
    assert attn(T=0, max_q=0, groups=None) == INVALID
    for args in ((0, 4, 2, 1, 4), (2, -1, 2, 1, 4), (2, 4, 0, 1, 4), (2, 4, 2, 1, 3), (2, 4, 2, -1, 4), (2, 4, 2, 65536, 4)):
        assert bx.ix_kv8_attn_shared_workspace_size(desc(), *args) == 0
    assert bx.ix_kv8_attn_shared_workspace_size(desc(), 2, 4, 2, 0, 4) == bx.ix_kv8_attn_workspace_size(desc(), 2, 4, 2, 4)
    assert attn(n_groups=0, groups=None, shared=None, o=None) == INVALID and attn(n_groups=0, groups=None, shared=None, T=0, max_q=0) == 0


def test_workspace_of_larger_batches():
    """One sized for the largest batch does for smaller ones."""
    for c in (desc(d=64), desc(d=128), desc(d=256)):
        last = 0
        for T, max_q in ((1, 1), (64, 1), (64, 64), (4096, 64), (4096, 4096), (50000, 4096)):
            n = bx.ix_kv8_attn_shared_workspace_size(c, 64, T, max_q, 3, 16)
            assert n >= last
            last = n


# ---- on the GPU --------------------------------------------------------------------------------

class Shared(Problem):
    """groups: [(shared tokens, [(new, tokens in all) of each sequence])]; a group of 0 shared tokens is none where `loose`."""

    def __init__(self, groups, page=16, h=2, d=64, G=2, seed=0, loose=False, before=0, **kw):
        lens = [x for _, g in groups for x in g]
        super().__init__([m for m, _ in lens], [n for _, n in lens], page, h, d, G, seed, **kw)
        ends = cumulative([len(g) for _, g in groups])
        given = [i for i, (n, _) in enumerate(groups) if n or not loose]
        assert given == list(range(given[0], given[0] + len(given))) if given else True
        self.shared = [groups[i][0] for i in given]
        self.groups = [ends[i] for i in given] + [ends[given[-1] + 1]] if given else []
        ref = self.p.ref
        for n, a, b in zip(self.shared, self.groups, self.groups[1:]):
            whole = n // page
            for i in range(a + 1, b):
                self.tables[i, :whole] = self.tables[a, :whole]
                if n % page and self.tables[a, whole] >= 0:
                    for x in "kv":
                        ref.codes[x][self.tables[i, whole], :, :n % page] = ref.codes[x][self.tables[a, whole], :, :n % page]
                        ref.scale[x][self.tables[i, whole]] = ref.scale[x][self.tables[a, whole]]

    def run(self, gate=False, q=None, max_q=None, out=None, n=None, s=None):
        import torch
        self.upload()
        q = bf(self.q_bits) if q is None else q
        o = torch.full((max(self.T, 1), self.h * self.G, self.d), float("nan"), dtype=torch.bfloat16, device="cuda")
        a = (self.p.cache, len(self.q_len), self.T, max_q or max(max(self.q_len), 1), ints(cumulative(self.q_len)), ints(self.kv_len),
             ints(self.tables), self.tables.shape[1])
        n = bx.ix_kv8_attn_shared_workspace_size(self.p.cache, *a[1:4], len(self.shared), self.h * self.G)
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")       # NaN, wherever it is read unwritten
        assert bx.ix_kv8_attn_shared(*a, len(self.shared), ints(self.groups) if self.groups else None, ints(self.shared) if self.groups else None, q,
                                     self.h * self.G, self.scale, bf(self.g_bits) if gate else None, o, ws, n, s) == 0
        return o.float().cpu().numpy()

    def both(self, **kw):
        got = self.run(**kw)
        self.check(got, gate=kw.get("gate", False))
        return got


def group(shared, *lens):
    """Sequences of (new, own tokens behind the shared ones, the new ones among them)."""
    return shared, [(m, shared + n) for m, n in lens]


LAYOUTS = [(16, 2, 64, 2), (32, 1, 128, 4), (64, 3, 128, 1), (128, 1, 256, 8), (16, 2, 256, 5), (64, 2, 64, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d,G", LAYOUTS)
@pytest.mark.parametrize("shared", [1, 15, 16, 64, 130, 1000])
def test_tokens(page, h, d, G, shared):
    """One token each of a few sequences behind shared ones of any length; the first has no token of its own but the new one."""
    Shared([group(shared, (1, 1), (1, 2), (1, 37), (1, 200))], page, h, d, G, shared).both(gate=shared % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d,G", LAYOUTS)
@pytest.mark.parametrize("n_seq", [2, 40, 130])
def test_many(page, h, d, G, n_seq):
    """Blocks of rows, in parts and whole, behind a long prefix that ends inside a page."""
    g = np.random.default_rng(n_seq)
    Shared([group(777, *[(1, int(n)) for n in g.integers(1, 90, n_seq)])], page, h, d, G, n_seq).both(gate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d,G", LAYOUTS)
def test_groups(page, h, d, G):
    """Groups of different sizes and lengths, one of one sequence, an empty one, one that shares nothing; drafts, prompts, and
    sequences without new tokens among them."""
    Shared([group(300, (1, 5), (4, 4), (0, 7)), group(64, (2, 130)), group(50), group(0, (1, 9), (30, 30)), group(1025, (0, 0), (1, 1), (3, 70)),
            group(17, (0, 3), (0, 0))], page, h, d, G, 5).both()


@pytest.mark.gpu
@pytest.mark.parametrize("page,h,d,G", LAYOUTS)
@pytest.mark.parametrize("new", [9, 70, 300])
def test_prompts(page, h, d, G, new):
    """Questions about one document: blocks of rows on both sides."""
    Shared([group(500, (new, new), (new // 2, new), (1, 1), (new, new + 77))], page, h, d, G, new).both(gate=True)


@pytest.mark.gpu
def test_sequences_of_no_group():
    """The groups are some of the batch, from its second sequence on."""
    p = Shared([group(0, (1, 40)), group(90, (1, 3), (2, 8)), group(33, (1, 1), (1, 30)), group(0, (1, 1), (20, 40))], loose=True)
    assert p.groups == [1, 3, 5]
    p.both()
    p = Shared([group(0, (1, 40), (3, 3))], loose=True)
    assert not p.groups
    p.both()


@pytest.mark.gpu
def test_many_groups():
    g = np.random.default_rng(6)
    Shared([group(int(n), *[(1, int(m)) for m in g.integers(1, 20, 1 + i % 3)]) for i, n in enumerate(g.integers(0, 120, 150))], h=1, G=4).both()


@pytest.mark.gpu
@pytest.mark.parametrize("n_groups", [2, 60, 300])
def test_many_sequences(n_groups):
    """More sequences and groups than are kept beside the kernel's rows, of more lengths than a wave has lanes."""
    g = np.random.default_rng(n_groups)
    each = 620 // n_groups
    Shared([group(int(n), *[(int(m > 2), int(m)) for m in g.integers(1, 20, each)]) for n in g.integers(0, 200, n_groups)], h=1, G=2).both()


@pytest.mark.gpu
@pytest.mark.parametrize("n_groups,each", [(100, 6), (20, 30), (70, 3)])
def test_groups_that_save_something_and_groups_that_do_not(n_groups, each):
    """Shared tokens from none to 12 tiles of them, in up to and over 64 groups, of up to and over 512 units."""
    g = np.random.default_rng(each)
    Shared([group(int(n), *[(1, int(m)) for m in g.integers(1, 30, each)]) for n in g.integers(0, 800, n_groups)], h=1, G=2).both()


@pytest.mark.gpu
def test_many_groups_of_many_rows():
    """Over 64 groups by blocks of 128 rows, whose parts are then cut by the room for them."""
    g = np.random.default_rng(3)
    Shared([group(int(n), (1, 9), (1, 1), (1, 30)) for n in g.integers(2500, 3500, 66)], page=128, h=1, d=64, G=48).both()


@pytest.mark.gpu
def test_thousands_of_sequences():
    """2,500 of one token each in 3 groups, 5,000 without new tokens among them."""
    g = np.random.default_rng(8)
    lens = [(int(i % 3 == 0), int(n)) for i, n in enumerate(g.integers(1, 5, 7500))]
    Shared([group(64, *lens[:3000]), group(0, *lens[3000:3100]), group(100, *lens[3100:])], h=1, G=1).both()


@pytest.mark.gpu
def test_sequences_longer_than_said():
    """Rows of sequences with more new tokens than max_q says are not written, those of the others are right."""
    for new, G in ((3, 2), (200, 8)):
        p = Shared([group(130, (1, 1), (new, new + 9), (2, 2))], h=2, G=G, seed=new)
        got = p.run(max_q=new - 1)
        assert np.isnan(got[1:1 + new]).all()
        got[1:1 + new] = p.run()[1:1 + new]
        p.check(got)


@pytest.mark.gpu
def test_as_without_groups():
    """Without groups the call is ix_kv8_attn; groups that share nothing, and groups of one sequence, are right."""
    lens = [(1, 300), (5, 90), (1, 1), (40, 700)]
    p = Shared([group(0, *lens)], loose=True)
    assert not p.groups and np.array_equal(p.both(), Problem.run(p))
    Shared([group(0, *lens)]).both()
    Shared([(n // 2, [(m, n)]) for m, n in lens]).both()


@pytest.mark.gpu
def test_lost_pages():
    """Shared pages without a place hide their tokens; where that is all a row could see beside its own, and where its own is lost."""
    for lost in ([0], [0, 1, 2, 3], [2]):
        p = Shared([group(64, (1, 1), (1, 20), (2, 40))])
        for i in range(3):
            p.tables[i, lost] = -1
        p.both()
    p = Shared([group(64, (1, 1), (1, 20), (2, 16))])
    p.tables[2, 4:] = p.p.ref.n_pages + 5
    p.tables[:, :4] = -1
    got = p.both()
    assert np.all(got[2:] == 0)                                 # of zeros, not of what the workspace held


@pytest.mark.gpu
def test_shared_tokens_that_are_new():
    """What the documentation rules out stays inside the cache and the outputs: more shared tokens than a sequence has."""
    p = Shared([group(64, (1, 1), (1, 20))])
    p.shared[0] = 200
    got = p.run()
    assert got.shape[0] == 2
    for n in (-5, 1 << 30):
        p.shared[0] = n
        p.run()
    for groups in ([0, 1 << 30], [-7, 2], [2, 0]):
        p.shared, p.groups = [64], groups
        p.run()
    p = Shared([group(64, *[(1, 20)] * 40)], G=16)
    for n in (3, 700):                                          # groups that overlap, over and over
        p.shared, p.groups = [64] * n, ([0, 40] * n)[:n + 1]
        p.run()


@pytest.mark.gpu
@pytest.mark.parametrize("scales", [(1e-30, 1.0), (1.0, 1e-30), (1e30, 1e-6), (0.0, 1.0), (1.0, 0.0)])
def test_scales_apart(scales):
    """Pages of shared and own tokens whose value scales lie far apart."""
    p = Shared([group(128, (1, 1), (1, 32), (3, 40))], v_std=1.0)
    ref = p.p.ref
    for x, at in zip(scales, (p.tables[0, :8], p.tables[:, 8:11])):
        at = at[at >= 0]
        ref.scale["v"][at] = np.float32(x) * ref.scale["v"][at] / np.float32(0.025)
    p.both()


@pytest.mark.gpu
def test_offsets_behind_the_first_row():
    """A part of a larger batch: rows before and behind are neither read nor written."""
    import torch
    p = Shared([group(100, (1, 1), (2, 30), (1, 9))], G=8, d=128)
    before, behind = 300, 50
    T = before + p.T + behind
    q = torch.full((T, p.h * p.G, p.d), float("nan"), dtype=torch.bfloat16, device="cuda")
    q[before:before + p.T] = bf(p.q_bits)
    p.upload()
    o = torch.full_like(q, 7.0)
    for max_q in (2, T):
        n = bx.ix_kv8_attn_shared_workspace_size(p.p.cache, 3, T, max_q, 1, p.h * p.G)
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
        o.fill_(7.0)
        assert bx.ix_kv8_attn_shared(p.p.cache, 3, T, max_q, ints(before + np.array(cumulative(p.q_len))), ints(p.kv_len), ints(p.tables),
                                     p.tables.shape[1], 1, ints(p.groups), ints(p.shared), q, p.h * p.G, p.scale, None, o, ws, n) == 0
        assert bool((o[:before] == 7).all()) and bool((o[before + p.T:] == 7).all())
        p.check(o[before:before + p.T].float().cpu().numpy())


@pytest.mark.gpu
def test_in_place_and_slices():
    """q as a slice of wider rows, and o in the memory of a packed q and of the gate."""
    import torch
    p = Shared([group(70, (1, 1), (4, 20), (1, 3))])
    wide = torch.zeros(p.T, p.h * p.G * p.d + 3, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:] = bf(p.q_bits).view(p.T, -1)
    want = p.run()
    assert np.array_equal(p.run(q=wide[:, 3:]), want)
    a = (p.p.cache, 3, p.T, 4, ints(cumulative(p.q_len)), ints(p.kv_len), ints(p.tables), p.tables.shape[1], 1, ints(p.groups), ints(p.shared))
    n = bx.ix_kv8_attn_shared_workspace_size(p.p.cache, 3, p.T, 4, 1, p.h * p.G)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    q = bf(p.q_bits)
    assert bx.ix_kv8_attn_shared(*a, q, p.h * p.G, p.scale, None, q, ws, n) == 0
    assert np.array_equal(q.float().cpu().numpy(), want)
    want, gate, q = p.run(gate=True), bf(p.g_bits), bf(p.q_bits)
    assert bx.ix_kv8_attn_shared(*a, q, p.h * p.G, p.scale, gate, gate, ws, n) == 0
    assert np.array_equal(gate.float().cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("G,d", [(2, 64), (8, 256)])
def test_captured(G, d):
    """Replays of a captured call with other lengths, groups and rows, eager calls on another stream and workspace between."""
    import torch
    p = Shared([group(400, *[(1, 100)] * 20)], h=2, d=d, G=G)
    p.upload()
    kv, groups, shared = ints(p.kv_len), ints([0, 20, 20]), ints([400, 0])
    cu, table, q = ints(range(21)), ints(p.tables), bf(p.q_bits)
    n = bx.ix_kv8_attn_shared_workspace_size(p.p.cache, 20, 20, 1, 2, 2 * G)
    ws = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for _ in "ab"]
    o = [torch.empty_like(q) for _ in "ab"]

    def call(i, s=None):
        assert bx.ix_kv8_attn_shared(p.p.cache, 20, 20, 1, cu, kv, table, table.shape[1], 2, groups, shared, q, 2 * G, p.scale, None, o[i],
                                     ws[i], n, s) == 0

    stream = torch.cuda.Stream()
    call(1, stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    for a, b, c, m in ((20, 400, 0, 500), (5, 100, 333, 420), (0, 0, 16, 17), (19, 399, 1, 480), (20, 0, 0, 31)):
        groups[1], shared[0], shared[1] = a, b, c
        kv.fill_(m)
        q.normal_()
        torch.cuda.synchronize()
        graph.replay()
        call(1, stream)
        torch.cuda.synchronize()
        assert torch.equal(o[0], o[1]) and bool(o[0].isfinite().all())
