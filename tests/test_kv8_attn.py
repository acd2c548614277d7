"""ix_kv8_attn against the attention of tests/kv8_ref.py in 64 bits, on the cache's own codes and scales.

Tolerance. Scores: q is rounded to 16 bits of its row's largest value, at most amax / 65278 a channel, so a
score is off by at most scale * amax / 65278 * sum|k| =: e1, and its 32-bit product, sum and exponential by
2^-22 (|s| + 16) log2(e)-wise, e2; p is within e1 + e2 relative of its value, rounded to fp16 for the values' product
(2^-11, or 2^-33 of the largest p where that is more), and summed in 32 bits over n tokens in blocks (the sum's
terms are rounded 2^-24 each, at most n / 16 + 64 of them in one chain). So
  |o - want| <= max|v| * (2 (e1 + e2) + 2^-11 + n 2^-32 + (n / 16 + 64) 2^-23) + 2^-8 |want| (bf16's half ulp of the result),
the factor 2 because numerator and denominator both move. A gate in (0, 1) only shrinks it."""
import ctypes

import numpy as np
import pytest

import baloon_amd as bx
from oracle import bf16
from tests import kv8_ref
from tests.test_kv8_cache import Pair, bf, cumulative, desc, ints, tables_for

INVALID = bx.HIP_ERROR_INVALID_VALUE
A = 1 << 20


def attn(c=None, n_seq=2, T=4, max_q=2, cu=A, kv=A, table=A, width=3, q=(A, 256), h_q=4, window=0, sinks=0, gate=None, o=A, ws=A,
         nbytes=1 << 40):
    r = [None if x is None else ctypes.byref(bx.Rows(*x)) for x in (q, gate)]
    return bx.lib().ix_kv8_attn(None if c == 0 else ctypes.byref(c or desc()), n_seq, T, max_q, cu, kv, table, width, r[0], h_q,
                                ctypes.c_float(1), window, sinks, r[1], o, ws, nbytes, None)


def test_refusals():
    assert attn(0) == INVALID
    for c in (desc(n_pages=0), desc(page=48), desc(h=0), desc(d=96), desc(k=None), desc(vs=None), desc(k=A + 4)):
        assert attn(c) == INVALID
    for kw in (dict(n_seq=0), dict(n_seq=65536), dict(T=-1), dict(max_q=0), dict(max_q=-1), dict(cu=None), dict(kv=None), dict(table=None),
               dict(width=0), dict(cu=A + 2), dict(h_q=0), dict(h_q=3), dict(h_q=-4), dict(window=-1), dict(window=(1 << 30) + 1),
               dict(sinks=-1), dict(o=None), dict(o=A + 1), dict(ws=None), dict(ws=A + 16), dict(q=None), dict(q=(None, 256)),
               dict(q=(A, 255)), dict(q=(A + 1, 256)), dict(gate=(None, 256)), dict(gate=(A, 255)), dict(gate=(A + 1, 256))):
        assert attn(**kw) == INVALID, kw
    need = bx.ix_kv8_attn_workspace_size(desc(), 2, 4, 2, 4)
    assert need > 0 and attn(nbytes=need - 1) == INVALID
    assert attn(T=0, max_q=0) == bx.HIP_SUCCESS
    for args in ((0, 4, 2, 4), (2, -1, 2, 4), (2, 4, 0, 4), (2, 4, 2, 3), (2, 4, 2, 0)):
        assert bx.ix_kv8_attn_workspace_size(desc(), *args) == 0
    assert bx.ix_kv8_attn_workspace_size(desc(d=96), 2, 4, 2, 4) == 0


# ---- on the GPU --------------------------------------------------------------------------------

class Problem:
    """A cache filled token by token in blocks through the reference, sequences of kv_len tokens whose last
    q_len are the queries'."""

    def __init__(self, q_len, kv_len, page=16, h=2, d=64, G=2, seed=0, q_std=2.0, v_std=1.0, spare=3):
        self.q_len, self.kv_len, self.h, self.d, self.G = list(q_len), list(kv_len), h, d, G
        n_pages = sum(-(-max(n, 0) // page) for n in kv_len) + spare
        self.p = Pair(n_pages, page, h, d, seed)
        g = self.p.g
        self.tables = tables_for(g, n_pages, [max(n, 0) for n in kv_len], page, max(-(-max(kv_len) // page), 1) + 1)
        ref = self.p.ref
        for n in "kv":                                           # codes and scales of pages that were appended to
            ref.codes[n][:] = np.clip(np.rint(g.normal(0, 40, ref.codes[n].shape)), -127, 127).astype(np.int8)
            ref.scale[n][:] = (g.uniform(0.5, 1.5, ref.scale[n].shape) * (v_std if n == "v" else 1.0) / 40).astype(np.float32)
        self.T = sum(q_len)
        self.q_bits, self.q = kv8_ref.normal_bf16(g, max(self.T, 1), h * G, d, std=q_std)
        self.g_bits, self.gate = kv8_ref.normal_bf16(g, max(self.T, 1), h * G, d)
        self.scale = d ** -0.5

    def upload(self):
        import torch
        c, s, t = self.p.ref.codes, self.p.ref.scale, self.p.t
        t[0].copy_(torch.from_numpy(c["k"].copy()))
        t[1].copy_(torch.from_numpy(np.ascontiguousarray(c["v"].swapaxes(2, 3))))
        t[2].copy_(torch.from_numpy(s["k"].copy()))
        t[3].copy_(torch.from_numpy(s["v"].copy()))

    def args(self, max_q=None):
        return (self.p.cache, len(self.q_len), self.T, max_q or max(max(self.q_len), 1), ints(cumulative(self.q_len)), ints(self.kv_len),
                ints(self.tables), self.tables.shape[1])

    def run(self, window=0, sinks=0, gate=False, q=None, scale=None, max_q=None, upload=True):
        import torch
        if upload:
            self.upload()
        a = self.args(max_q)
        q = bf(self.q_bits) if q is None else q
        o = torch.full((max(self.T, 1), self.h * self.G, self.d), float("nan"), dtype=torch.bfloat16, device="cuda")
        n = bx.ix_kv8_attn_workspace_size(self.p.cache, *a[1:4], self.h * self.G)
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")       # NaN, wherever it is read unwritten
        assert bx.ix_kv8_attn(*a, q, self.h * self.G, self.scale if scale is None else scale, window, sinks,
                              bf(self.g_bits) if gate else None, o, ws, n) == 0
        return o.float().cpu().numpy()

    def check(self, got, window=0, sinks=0, gate=False, scale=None):
        scale = self.scale if scale is None else scale
        at = 0
        for b, (m, n) in enumerate(zip(self.q_len, self.kv_len)):
            n = max(n, 0)
            k, has = self.p.ref.tokens("k", n, self.tables[b])
            v, _ = self.p.ref.tokens("v", n, self.tables[b])
            seen = kv8_ref.seen_by(m, n, has, window, sinks)
            k[~seen.any(0)] = 0
            v[~seen.any(0)] = 0
            q = self.q[at:at + m]
            want = kv8_ref.attend(q, n, k, v, seen, scale, self.gate[at:at + m] if gate else None)
            if m and n:
                amax = np.abs(q).max(2, keepdims=True)
                sum_k = np.abs(k).sum(2).max()
                e1 = abs(scale) * amax / 65278 * sum_k
                e2 = 2.0 ** -22 * (abs(scale) * amax * sum_k + 16) * 1.5
                tol = np.abs(v).max() * (2 * (e1 + e2) + 2.0 ** -11 + n * 2.0 ** -32 + (n / 16 + 64) * 2.0 ** -23) + 2.0 ** -8 * np.abs(want)
                near = np.abs(got[at:at + m] - want) <= tol
                assert near.all(), (b, np.argwhere(~near)[:5], got[at:at + m][~near][:5], want[~near][:5], tol[~near][:5])
            else:
                assert np.all(got[at:at + m] == 0), b
            at += m

    def both(self, **kw):
        max_q = kw.pop("max_q", None)
        self.check(self.run(max_q=max_q, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("h,G", [(1, 1), (2, 8), (3, 5), (2, 17)])
def test_single_tokens(d, page, h, G):
    """One new token a sequence, of lengths around the pages' and tiles' ends."""
    kv = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300, 1000]
    Problem([1] * len(kv), kv, page, h, d, G, seed=d + page + G).both(gate=G == 8)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kv", [1, 64, 5000, 40001])
def test_one_sequence(d, kv):
    """One sequence over all the workgroups."""
    Problem([1], [kv], 16, 2, d, 8, seed=kv).both()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 4, 8])
def test_drafts_and_prompts(d, G):
    """Several new tokens: windows of drafts, prompts from the start and behind cached tokens, mixed in a batch with
    sequences that have none."""
    Problem([4, 0, 7, 1, 3, 8], [4, 50, 90, 1, 300, 1025], 32, 2, d, G, seed=G).both(gate=True)
    Problem([100, 1, 0, 333, 64, 5], [100, 700, 3, 400, 1000, 5], 16, 2, d, G, seed=G + 1).both(gate=G == 4)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("G", [1, 3, 8])
def test_long_prompts(d, page, G):
    """Batches of enough rows for blocks of 256: prompts from the start and behind cached tokens, of lengths around the
    blocks', with single tokens and empty sequences among them."""
    n = 64 * 256 // (8 * G)
    q = [n // 2 + 5, 1, 0, 256 // G + 1, n // 3, 64, 256 // G, n // 6 + 40]
    kv = [q[0], 700, 3, q[3] + 200, q[4] + 77, 64, q[6] + 1, q[7] + 1000]
    Problem(q, kv, page, 8, d, G, seed=G).both(gate=G == 3)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 3), (300, 200), (64, 0), (2000, 4), (5, 2 ** 31 - 1)])
def test_long_prompts_in_a_window(d, window, sinks):
    Problem([900, 3, 700], [900, 2000, 1900], 16, 8, d, 2, seed=window).both(window=window, sinks=sinks)
    Problem([3000], [3100], 64, 8, 64, 1, seed=sinks % 999, q_std=1.0).both(window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_prompts_that_see_little(d):
    """Pages that are gone, tokens before the start, scales that are not numbers in hidden places, and edges of scales and
    scores, in blocks of 256 rows."""
    P = Problem([1500, 700, 40], [1400, 720, 30], 16, 8, d, 2, seed=1, spare=8)
    ref = P.p.ref
    P.tables[0, 5:9] = [-1, 1 << 30, -7, -1]
    P.tables[1, :] = -5
    used = set(P.tables[(P.tables >= 0) & (P.tables < ref.n_pages)].tolist())
    for i in set(range(ref.n_pages)) - used:
        for n in "kv":
            ref.codes[n][i] = -128
            ref.scale[n][i] = [np.nan, np.inf][i % 2]
    for n in "kv":
        ref.codes[n][P.tables[0, 2]] = 0
        ref.scale[n][P.tables[0, 2]] = 0
        for p in range(20, 40):
            ref.scale[n][P.tables[0, p]] *= np.float32(10.0 ** (p % 5 - 3))
    ref.scale["k"][P.tables[0, 60:]] *= 30
    P.q[100:200] = 0
    P.q[300:400, :, 5] *= 50
    P.q_bits = bf16.from_f32(P.q)
    P.q = bf16.to_f32(P.q_bits)
    P.both(gate=True)
    P.both(scale=-0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (63, 0), (64, 100), (100, 17), (300, 1), (5000, 4), (7, 2 ** 31 - 1),
                                         (2 ** 30, 4)])
def test_window_and_sinks(d, window, sinks):
    kv = [1, 5, 64, 65, 130, 200, 333, 1000]
    Problem([1] * len(kv), kv, 16, 2, d, 4, seed=window % 1000).both(window=window, sinks=sinks)
    Problem([3, 60, 200, 130], [500, 60, 420, 131], 64, 1, d, 5, seed=sinks % 999).both(window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq", [1, 2, 63, 64, 65, 200, 1000])
def test_many_sequences(n_seq):
    g = np.random.default_rng(n_seq)
    kv = [int(x) for x in g.integers(1, 200, n_seq)]
    q = [int(min(n, x)) for n, x in zip(kv, g.integers(0, 3, n_seq))]
    q[0] = 1
    Problem(q, kv, 16, 1, 64, 2, seed=n_seq, spare=40).both()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 256])
def test_rows_that_see_nothing(d):
    """No tokens at all, tokens before the sequence's start, pages that are gone: zeros, whatever lies in the cache."""
    P = Problem([1, 3, 2, 1, 40], [0, 1, 40, 20, 10], 16, 2, d, 4, seed=1)
    P.tables[2, :2] = [-1, 1 << 30]                             # of 40 tokens the last 8 are there
    P.tables[3, :] = -5
    P.both(gate=True)
    P.both(window=4, sinks=2)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q", [1, 3, 150])
def test_hidden_values(d, q):
    """Scales that are infinite or not numbers, and the largest codes, in hidden places: pages of nobody, entries behind the
    last page, tokens that the window hides."""
    P = Problem([q] * 3, [q, q + 200, q + 555], 16, 2, d, 4, seed=7, spare=8)
    ref = P.p.ref
    used = set(P.tables[P.tables >= 0].tolist())
    for i in set(range(ref.n_pages)) - used:
        for n in "kv":
            ref.codes[n][i] = -128
            ref.scale[n][i] = [np.nan, np.inf][i % 2]
    spare = min(set(range(ref.n_pages)) - used)
    P.tables[P.tables < 0] = spare                               # entries behind the last page
    P.both()
    P.tables[2, 2:(555 - 70) // 16] = spare                      # what a window of 64 and 17 sinks hides
    P.tables[1, 2:(200 - 70) // 16] = spare
    P.both(window=64, sinks=17)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 200])
def test_scales_and_scores_at_the_edges(q):
    """Pages of zeros, pages of very different scales, scores so large that one token decides, q of zeros and outliers."""
    P = Problem([q] * 5, [q + 300] * 5, 16, 1, 128, 4, seed=3)
    ref, t = P.p.ref, P.tables
    for n in "kv":
        for p in (0, 3, 4, 18):
            ref.codes[n][t[0, p]] = 0
            ref.scale[n][t[0, p]] = 0
        for p in range(19):
            ref.scale[n][t[1, p]] *= np.float32(10.0 ** (p % 5 - 3))
    ref.scale["k"][t[2]] *= 100                                  # of row 2's pages: scores of thousands
    cu = cumulative(P.q_len)
    P.q[cu[3]:cu[4]] = 0
    P.q[cu[4]:cu[5], :, 5] *= 50
    P.q_bits = bf16.from_f32(P.q)
    P.q = bf16.to_f32(P.q_bits)
    P.both()
    P.both(scale=-0.05)
    P.both(scale=0.0)


@pytest.mark.gpu
def test_flat_long_context_with_a_sink():
    """One token takes half of the weight, 60,000 share the rest: each of theirs is 2^-16 of the largest."""
    n, d = 60000, 64
    P = Problem([1], [n], 64, 1, d, 1, seed=5, q_std=1.0)
    ref = P.p.ref
    P.q[:] = 0
    P.q[:, :, 0] = 8
    P.q_bits = bf16.from_f32(P.q)
    ref.codes["k"][:, :, :, 0] = 0
    first = P.tables[0, 0]
    ref.scale["k"][:] = np.float32(1 / 127)
    ref.codes["k"][first, 0, 0, 0] = 127
    ref.codes["v"][:] = np.abs(ref.codes["v"])
    ref.codes["v"][first, 0, 0] = 0
    P.both(scale=float(np.log(n) / 8))
    got = P.run(scale=float(np.log(n) / 8))
    assert got.min() > 0.1                                       # the small ones count


@pytest.mark.gpu
def test_rows_not_finite_stay_alone():
    """A query that is not a number spoils its own row only."""
    for q in (1, 130, 600):
        P = Problem([q, q], [q + 70, q + 9], 16, 2, 128, 8, seed=q)
        clean = P.run()
        P.q[0, 3] = np.nan
        P.q[1, 15, 7] = np.inf
        P.q_bits = bf16.from_f32(P.q)
        got = P.run()
        for t, h in ((0, 3), (1, 15)):
            assert np.isnan(got[t, h]).any()
            got[t, h] = clean[t, h]
        assert np.array_equal(got, clean)


@pytest.mark.gpu
def test_operands_and_repeats():
    """q and gate as slices of wider rows, of odd strides, o over q; the same bits each time."""
    import torch
    for q in ([1, 1, 1], [5, 200, 3], [5, 2200, 3]):
        P = Problem(q, [40, 900 if q[1] < 900 else 2300, 3], 16, 2, 128, 4, seed=4)
        n, d = 8, 128
        want = P.run(gate=True)
        P.check(want, gate=True)
        assert np.array_equal(P.run(gate=True), want)
        a = P.args()
        size = bx.ix_kv8_attn_workspace_size(P.p.cache, *a[1:4], n)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        wide = torch.zeros(P.T, 3, n, d, dtype=torch.bfloat16, device="cuda")
        wide[:, 1], wide[:, 2] = bf(P.q_bits), bf(P.g_bits)
        odd = torch.zeros(P.T, 2 * n * d + 3, dtype=torch.bfloat16, device="cuda")
        odd[:, 1:n * d + 1], odd[:, n * d + 2:-1] = bf(P.q_bits).view(P.T, -1), bf(P.g_bits).view(P.T, -1)
        own = bf(P.q_bits)
        for rows, gate, o in ((wide[:, 1], wide[:, 2], None), (odd[:, 1:n * d + 1], odd[:, n * d + 2:-1], None), (own, bf(P.g_bits), own)):
            o = torch.empty(P.T, n, d, dtype=torch.bfloat16, device="cuda") if o is None else o
            assert bx.ix_kv8_attn(*a, rows, n, P.scale, 0, 0, gate, o, ws, size) == 0
            assert np.array_equal(o.float().cpu().numpy(), want)
        off = torch.empty(P.T * n * d + 1, dtype=torch.bfloat16, device="cuda")[1:]
        assert bx.ix_kv8_attn(*a, bf(P.q_bits), n, P.scale, 0, 0, bf(P.g_bits), off, ws, size) == 0
        assert np.array_equal(off.float().cpu().numpy().reshape(want.shape), want)


@pytest.mark.gpu
def test_graph_replays_with_other_lengths():
    """A captured call, replayed after the lengths and pages have changed, equals the eager call each time."""
    import torch
    P = Problem([1] * 4, [700, 3, 65, 1500], 16, 2, 128, 4, seed=6)
    P.upload()
    a = P.args()
    cu, kv, table = a[4:7]
    q = bf(P.q_bits)
    n = bx.ix_kv8_attn_workspace_size(P.p.cache, *a[1:4], 8)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    o, e = (torch.empty(4, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in "ab")
    call = lambda out: bx.ix_kv8_attn(P.p.cache, 4, 4, 1, cu, kv, table, a[7], q, 8, P.scale, 0, 0, None, out, ws, n)
    assert call(o) == 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert call(o) == 0
    for lens in ([700, 3, 65, 1500], [1, 1, 1, 1], [64, 2, 17, 1499], [0, 3, 40, 1024]):
        kv.copy_(ints(lens))
        o.zero_()
        g.replay()
        assert call(e) == 0
        torch.cuda.synchronize()
        assert torch.equal(o, e)
        P.kv_len = lens
        P.check(o.float().cpu().numpy())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    import torch
    n_pages, page, h, d = 700_000, 16, 2, 256
    P = Problem([1, 2, 2100], [40, 300, 2200], page, h, d, 4, seed=9)
    big = [torch.empty(n_pages, h, page, d, dtype=torch.int8, device="cuda"), torch.empty(n_pages, h, d, page, dtype=torch.int8, device="cuda")]
    big += [torch.empty(n_pages, h, device="cuda") for _ in "kv"]
    P.upload()
    m = P.p.ref.n_pages
    for t, x in zip(big, P.p.t):
        t[n_pages - m:].copy_(x)
    a = list(P.args())
    a[0] = bx.kv8_cache(*big)
    a[6] = torch.where(a[6] >= 0, a[6] + (n_pages - m), -1).to(torch.int32)
    o = torch.empty(P.T, h * 4, d, dtype=torch.bfloat16, device="cuda")
    n = bx.ix_kv8_attn_workspace_size(a[0], *a[1:4], h * 4)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert bx.ix_kv8_attn(*a, bf(P.q_bits), h * 4, P.scale, 0, 0, None, o, ws, n) == 0
    P.check(o.float().cpu().numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("d,page", [(64, 16), (64, 128), (128, 32), (128, 64), (256, 16), (256, 128)])
def test_blocks_in_parts(d, page):
    """So few blocks of rows that several workgroups share one: each block's parts are joined, those in which nothing is
    seen among them, and blocks that are too short for parts stand beside them."""
    P = Problem([256], [256 + 2900], page, 4, d, 8, seed=d + page)
    P.both(gate=True)
    P.both(window=1111, sinks=70)
    got = P.run()
    assert np.array_equal(P.run(), got)
    P = Problem([1, 140, 3, 0, 145, 37, 20], [900, 1500, 70, 40, 145, 2000, 10], page, 4, d, 8, seed=d * page)
    P.tables[1, :1100 // page] = -1                              # parts without a token
    P.tables[5, 700 // page:] = -1
    P.both()
    P.both(window=64, sinks=129, gate=True)
    P.both(window=1200, sinks=0, max_q=3000)


@pytest.mark.gpu
def test_blocks_in_parts_of_many_sequences():
    """More sequences than lanes, blocks among them from the first to the last."""
    q = [1 + 7 * (i % 5 == 0) for i in range(150)]
    q[0], q[63], q[64], q[149] = 70, 65, 33, 90
    P = Problem(q, [n + 37 * i % 600 for i, n in enumerate(q)], 16, 2, 256, 8, seed=11)
    P.both()


@pytest.mark.gpu
@pytest.mark.parametrize("n,h,width", [(1, 1024, 1 << 22), (70, 64, 1 << 20)])
def test_tables_with_places_for_more_than_32_bits_of_tiles(n, h, width):
    """The same bits with a table of so many places that counts of tiles could pass 32 bits."""
    import torch
    P = Problem([1 + i % 3 for i in range(n)], [3 + (41 * i) % 150 for i in range(n)], 16, h, 64, 1, seed=n)
    want = P.run()
    P.check(want)
    wide = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    wide[:, :P.tables.shape[1]] = ints(P.tables)
    c, b, T, max_q, cu, kv, _, _ = P.args()
    size = bx.ix_kv8_attn_workspace_size(c, b, T, max_q, h)
    ws, o = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(T, h, 64, dtype=torch.bfloat16, device="cuda")
    assert bx.ix_kv8_attn(c, b, T, max_q, cu, kv, wide, width, bf(P.q_bits), h, P.scale, 0, 0, None, o, ws, size) == 0
    assert np.array_equal(o.float().cpu().numpy(), want)


def test_workspace_sizes():
    """Of the sizes only: single tokens need little, and any batch a bounded size."""
    for d, few, most in ((64, 5, 38), (128, 9, 74), (256, 17, 81)):
        c = desc(h=8, d=d)
        assert bx.ix_kv8_attn_workspace_size(c, 1, 1, 1, 8) == bx.ix_kv8_attn_workspace_size(c, 500, 500, 1, 64) <= few << 20
        for n, T, max_q in ((1, 1 << 20, 1 << 20), (1, 512, 512), (64, 64 * 512, 512), (65535, 1 << 20, 4000), (3, 130, 100)):
            assert 0 < bx.ix_kv8_attn_workspace_size(c, n, T, max_q, 64) <= most << 20


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[3, 2, 1], [200, 1, 0], [0, 0, 256], [90, 90, 90]])
def test_offsets_that_end_before_the_rows(lens):
    """Room for 256 rows a sequence, as a captured call keeps it, of which the offsets use fewer: the rest is not written."""
    import torch
    P = Problem(lens, [n + 700 for n in lens], 16, 4, 256, 8, seed=sum(lens))
    P.upload()
    c, n, T, _, cu, kv, table, width = P.args()
    room = 3 * 256
    q = torch.zeros(room, 32, 256, dtype=torch.bfloat16, device="cuda")
    q[:T] = bf(P.q_bits)[:T]
    o = torch.full_like(q, 7)
    size = bx.ix_kv8_attn_workspace_size(c, n, room, 256, 32)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    assert bx.ix_kv8_attn(c, n, room, 256, cu, kv, table, width, q, 32, P.scale, 0, 0, None, o, ws, size) == 0
    P.check(o[:T].float().cpu().numpy())
    assert bool((o[T:] == 7).all())
