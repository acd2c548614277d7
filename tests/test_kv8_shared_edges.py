"""ix_kv8_attn_shared and ix_kv8_append_rope where they can go wrong beside lengths and layouts: hidden places, rows that are not
finite, scores and scales at the edges, many heads, tokens before position 0, caches of more than 2^32 bytes, memory at odd
addresses, workspaces that are used again. Tolerances as in tests/test_kv8_shared.py."""
import numpy as np
import pytest

import baloon_amd as bx
from oracle import bf16
from tests.test_kv8_cache import bf, cumulative, ints
from tests.test_kv8_shared import Shared, group

pytestmark = pytest.mark.gpu
SHAPES = [(64, 2), (128, 4), (256, 8)]
# 2 and 40 sequences: rows by 16; 40 behind 5,000 tokens: by 128
GROUPS = [(2, 200), (40, 200), (40, 5000)]


def of(n, shared, d, G, new=1, **kw):
    g = np.random.default_rng(n + shared + d)
    return Shared([group(shared, *[(new, int(m) + new) for m in g.integers(0, 90, n)]), group(0, (new, new + 40))], d=d, G=G, **kw)


@pytest.mark.parametrize("d,G", SHAPES)
@pytest.mark.parametrize("n,shared", GROUPS)
def test_hidden_places(d, G, n, shared):
    """Scales that are infinite or not numbers in pages of nobody, which also stand behind the tables' last pages, and in what the
    others of a group name for shared tokens that are read through the first one's table."""
    p = of(n, shared, d, G, spare=8)
    ref = p.p.ref
    used = set(p.tables[p.tables >= 0].tolist())
    free = sorted(set(range(ref.n_pages)) - used)
    for i in free:
        for x in "kv":
            ref.codes[x][i] = -128
            ref.scale[x][i] = [np.nan, np.inf][i % 2]
    p.tables[p.tables < 0] = free[0]
    p.both(gate=True)


@pytest.mark.parametrize("d,G", SHAPES)
@pytest.mark.parametrize("n,shared", GROUPS)
def test_rows_not_finite_stay_alone(d, G, n, shared):
    """A query that is not a number spoils its own row only, not those of other sequences beside it. These keep the tolerance, not
    their bits: 16 rows' references follow their maxima together, and where they do is where p is rounded differently."""
    p = of(n, shared, d, G)
    clean, q = p.run(), p.q.copy()
    p.q[0, 1] = np.nan
    p.q[n - 1, 2 * G - 1, 7] = np.inf
    p.q_bits = bf16.from_f32(p.q)
    got = p.run()
    for t, h in ((0, 1), (n - 1, 2 * G - 1)):
        assert np.isnan(got[t, h]).any()
        got[t, h] = clean[t, h]
    p.q = q
    p.check(got)


@pytest.mark.parametrize("d,G", SHAPES)
@pytest.mark.parametrize("n,shared", GROUPS)
def test_scales_and_scores_at_the_edges(d, G, n, shared):
    """Shared pages of zeros, pages of very different scales, scores so large that one token decides, queries of zeros and with
    outliers; negative and no scale of scores."""
    p = of(n, shared, d, G)
    ref, t = p.p.ref, p.tables
    for x in "kv":
        ref.codes[x][t[0, [0, 3]]] = 0
        ref.scale[x][t[0, [0, 3]]] = 0
        for i in range(5, 12):
            ref.scale[x][t[0, i]] *= np.float32(10.0 ** (i % 5 - 3))
    ref.scale["k"][t[1, shared // 16:][t[1, shared // 16:] >= 0]] *= 100
    p.q[0] = 0
    p.q[1, :, 5] *= 50
    p.q_bits = bf16.from_f32(p.q)
    p.q = bf16.to_f32(p.q_bits)
    for p.scale in (d ** -0.5, -0.05, 0.0):
        p.both()


@pytest.mark.parametrize("h,G,d", [(1, 160, 64), (2, 33, 128), (1, 128, 256), (3, 17, 64)])
@pytest.mark.parametrize("new", [1, 3])
def test_many_heads(h, G, d, new):
    Shared([group(200, (new, 5), (new, 40), (new, 3)), group(0, (new, 70))], h=h, G=G, d=d).both(gate=True)


@pytest.mark.parametrize("d,G", SHAPES)
def test_tokens_before_position_0(d, G):
    """More new tokens than there are in all: the first ones have no place and see nothing."""
    Shared([group(0, (9, 5), (1, 0)), group(70, (2, 2), (1, 9)), group(0, (40, 33), (3, 3))], d=d, G=G).both()


@pytest.mark.parametrize("d,G", SHAPES)
def test_the_same_bits_each_time(d, G):
    for n, shared in GROUPS:
        p = of(n, shared, d, G, new=2)
        first = p.run(gate=True)
        for _ in range(3):
            assert np.array_equal(p.run(gate=True), first)


def test_odd_addresses():
    """q, gate and o at any even address, rows of odd strides."""
    import torch
    p = of(5, 300, 128, 4)
    want = p.run(gate=True)

    def odd(bits):
        wide = torch.zeros(p.T, p.h * p.G * p.d + 1, dtype=torch.bfloat16, device="cuda")
        wide[:, 1:] = bf(bits).view(p.T, -1)
        return wide[:, 1:]

    a = (p.p.cache, len(p.q_len), p.T, 1, ints(cumulative(p.q_len)), ints(p.kv_len), ints(p.tables), p.tables.shape[1], len(p.shared), ints(p.groups),
         ints(p.shared))
    n = bx.ix_kv8_attn_shared_workspace_size(p.p.cache, *a[1:4], a[8], p.h * p.G)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    for shift in (1, 3, 4):
        o = torch.full((want.size + shift + 9,), 7.0, dtype=torch.bfloat16, device="cuda")
        assert bx.ix_kv8_attn_shared(*a, odd(p.q_bits), p.h * p.G, p.scale, odd(p.g_bits), o[shift:], ws, n) == 0
        got = o.float().cpu().numpy()
        assert np.array_equal(got[shift:shift + want.size], want.ravel()) and np.all(got[:shift] == 7) and np.all(got[shift + want.size:] == 7)


def test_graphs_that_share_a_workspace():
    """Two captured batches of different sizes, replayed in turn on one stream with one workspace sized for the larger."""
    import torch
    ps = [of(40, 1500, 128, 4), of(3, 900, 128, 4, new=5)]
    sizes = [bx.ix_kv8_attn_shared_workspace_size(p.p.cache, 41, p.T, max(p.q_len), 2, 8) for p in ps]
    most = bx.ix_kv8_attn_shared_workspace_size(ps[0].p.cache, 41, max(p.T for p in ps), 5, 2, 8)
    assert most >= max(sizes)
    ws = torch.full((most,), 0xFF, dtype=torch.uint8, device="cuda")
    graphs, outs, wants, held = [], [], [], []
    for p in ps:
        wants.append(p.run())
        p.upload()
        q = bf(p.q_bits)
        o = torch.empty_like(q)
        held.append((p.p.cache, len(p.q_len), p.T, max(p.q_len), ints(cumulative(p.q_len)), ints(p.kv_len), ints(p.tables), p.tables.shape[1], 2,
                     ints(p.groups), ints(p.shared), q, 8, p.scale, None, o, ws, most))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert bx.ix_kv8_attn_shared(*held[-1]) == 0
        graphs.append(graph)
        outs.append(o)
    for i in range(12):
        outs[i % 2].fill_(7.0)
        graphs[i % 2].replay()
        assert np.array_equal(outs[i % 2].float().cpu().numpy(), wants[i % 2]), i


def test_caches_of_more_than_32_bits():
    """The same batch in the first and in the last pages of a cache of 4.6 GB of codes: appended with positions and read by the attention,
    the same bits."""
    import torch
    page, h, d, G, n_pages = 128, 2, 256, 8, 70_000
    cache = bx.kv8_cache(torch.empty(n_pages, h, page, d, dtype=torch.int8, device="cuda"), torch.empty(n_pages, h, d, page, dtype=torch.int8, device="cuda"),
                         torch.empty(n_pages, h, device="cuda"), torch.empty(n_pages, h, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(2)
    freq = bx.rope_freq(d)[0].cuda()
    r = bx.rope(freq, norm=torch.rand(d, generator=g, device="cuda") + 0.5)
    T = 1500
    q, k, v = (torch.randn(T, n, d, generator=g, device="cuda").bfloat16() for n in (h * G, h, h))
    one = [torch.randn(6, n, d, generator=g, device="cuda").bfloat16() for n in (h * G, h, h)]
    width, results = 16, []
    need = bx.ix_kv8_attn_shared_workspace_size(cache, 6, 6, 1, 1, h * G)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    for at in (0, n_pages - 40):
        table = torch.full((6, width), -1, dtype=torch.int32, device="cuda")
        table[:, :11] = torch.arange(at, at + 11, dtype=torch.int32)             # 11 whole pages of the first 1,408 tokens
        table[:, 11] = torch.arange(at + 11, at + 17, dtype=torch.int32)
        cu, qt = ints([0, T]), torch.empty_like(q)
        assert bx.ix_kv8_append_rope(cache, 1, T, cu, ints([T]), table, width, k, v, r, q, h * G, r, qt) == 0
        for t in cache.tensors:                                                  # the page that they end in, for each
            t[at + 12:at + 17] = t[at + 11].clone()
        kv, cu = ints([T + 1] * 6), ints(range(7))
        turned, o = torch.empty_like(one[0]), torch.empty_like(one[0])
        assert bx.ix_kv8_append_rope(cache, 6, 6, cu, kv, table, width, one[1], one[2], r, one[0], h * G, r, turned) == 0
        assert bx.ix_kv8_attn_shared(cache, 6, 6, 1, cu, kv, table, width, 1, ints([0, 6]), ints([T]), turned, h * G, d ** -0.5, None, o, ws, need) == 0
        alone = torch.empty_like(o)
        n = bx.ix_kv8_attn_workspace_size(cache, 6, 6, 1, h * G)
        assert bx.ix_kv8_attn(cache, 6, 6, 1, cu, kv, table, width, turned, h * G, d ** -0.5, 0, 0, None, alone, torch.empty(n, dtype=torch.uint8, device="cuda"), n) == 0
        assert (o.float() - alone.float()).abs().max() <= 2.0 ** -7 * alone.abs().max()
        results.append((qt, turned, o, alone, *(t[at:at + 17, :].clone() for t in cache.tensors[:1]), *(t[at:at + 17].clone() for t in cache.tensors[2:])))
    assert all(torch.equal(a, b) for a, b in zip(*results))
