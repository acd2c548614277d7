"""AttnLayer with rotary positions, and with slots that were forked from one prompt: appends that turn, the cache and the attention
behind shared tokens as they are used together; and the hybrid stack's continuations of one prompt."""
import numpy as np
import pytest

import baloon_amd as bx
from tests import kv8_ref
from tests.test_attn_layer_calls import rows
from tests.test_kv8_cache import cumulative, ints

pytestmark = pytest.mark.gpu


def ropes(g, d, rot=None):
    """Descriptions for queries and for keys, which share their frequencies and have norms of their own."""
    import torch
    freq = bx.rope_freq(rot or d, 1e4)[0].cuda()
    return [bx.rope(freq, norm=torch.rand(d, generator=g, device="cuda") + 0.5) for _ in "qk"]


def drawn(g, T, h_q, h_kv, d):
    return [rows(g, T, h, d) for h in (h_q, h_kv, h_kv, h_q)]


def turned(layer, lens, q):
    """The queries of a call that has been made, as ix_rope_rows turns them."""
    import torch
    if layer.rope is None:
        return q
    y = torch.empty_like(q)
    assert bx.ix_rope_rows(layer.rope, layer.n_slots, q.shape[0], ints(cumulative(lens)), layer.kv_len, q, layer.h_q, layer.d, y) == 0
    return y


def check(layer, lens, q, z, got):
    """got against the attention in 64 bits over the codes that the table names, queries as they were turned to bf16. The tolerance is
    that of the layer's own test: 2^-8 of the result and 2^-9 of the largest value."""
    q, z, got = (t.double().cpu().numpy() for t in (turned(layer, lens, q), z, got))
    t = [x.cpu().numpy() for x in layer.cache.tensors]
    table, length, page, cu = layer.table.cpu().numpy(), layer.kv_len.tolist(), layer.cache.page, cumulative(lens)
    for b, m in enumerate(lens):
        if m == 0:
            continue
        at = np.arange(length[b])
        id = table[b, at // page]
        k = t[0][id, :, at % page].astype(np.float64) * t[2][id][:, :, None]
        v = t[1][id, :, :, at % page].astype(np.float64) * t[3][id][:, :, None]
        s = slice(cu[b], cu[b + 1])
        want = kv8_ref.attend(q[s], length[b], k, v, kv8_ref.seen_by(m, length[b], np.ones(length[b], bool), 0, 0), layer.scale, z[s])
        assert np.all(np.abs(got[s] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * np.abs(v).max()), b


@pytest.mark.parametrize("d,rot", [(64, 64), (128, 32), (256, 64)])
def test_positions(d, rot):
    """The layer with positions is the plain one on rows that ix_rope_rows has turned, bit for bit; also where o is the memory of
    q or of the gate."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(d)
    rq, rk = ropes(g, d, rot)
    layer = bx.AttnLayer(3, 300, 4, 2, d, 16, rope=rq, rope_k=rk)
    other = bx.AttnLayer(3, 300, 4, 2, d, 16)
    for i, lens in enumerate([(37, 0, 200), (1, 1, 1), (4, 4, 4), (1, 1, 1), (0, 50, 2)]):
        T, cu = sum(lens), ints(cumulative(lens))
        q, k, v, z = drawn(g, T, 4, 2, d)
        qt, kt, kv = torch.empty_like(q), torch.empty_like(k), other.kv_len + ints(lens)
        assert bx.ix_rope_rows(rq, 3, T, cu, kv, q, 4, d, qt) == 0 and bx.ix_rope_rows(rk, 3, T, cu, kv, k, 2, d, kt) == 0
        want = other.prefill(cu, max(lens), qt, kt, v, z)
        o = (None, q, z)[i % 3]
        got = layer.decode(q, k, v, z, o) if lens == (1, 1, 1) else layer.prefill(cu, max(lens), q, k, v, z, o)
        assert torch.equal(got, want), i
        assert all(torch.equal(a, b) for a, b in zip(layer.cache.tensors, other.cache.tensors)), i


@pytest.mark.parametrize("own_pages", [True, False])
@pytest.mark.parametrize("h_q,h_kv,d,page", [(4, 2, 64, 32), (8, 1, 256, 16), (6, 2, 128, 64)])
def test_forks(own_pages, h_q, h_kv, d, page):
    """Two forks of a batch beside slots of their own: tokens, drafts, a prompt for one, a release and another fork."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(h_q + page)
    rq, rk = ropes(g, d)
    layer = bx.AttnLayer(8, 400, h_q, h_kv, d, page, None if own_pages else 8 * -(-400 // page), rope=rq, rope_k=rk, max_forks=2, worth=0)
    if not own_pages:
        layer.table.copy_(torch.randperm(layer.cache.n_pages).view(8, -1))
    own = layer.table.clone()

    def step(*lens):
        rows = drawn(g, sum(lens), h_q, h_kv, d)
        one = all(m == 1 for m in lens)
        got = layer.decode(*rows) if one else layer.prefill(ints(cumulative(lens)), max(lens), *rows)
        check(layer, lens, rows[0], rows[3], got)

    step(20, 133, 0, 0, 3, 300, 7, 0)
    layer.fork(1, 3, 133)
    layer.fork(5, 3, 257)                                       # of 300 tokens that it holds
    assert layer.kv_len.tolist() == [20, 133, 133, 133, 3, 300, 257, 257]
    assert len(set(layer.table[1:4, 133 // page].tolist())) == 3 and len(set(layer.table[5:, 0].tolist())) == 1
    for _ in range(3):
        step(*[1] * 8)
    step(4, 4, 0, 2, 4, 4, 4, 4)
    layer.kv_len -= ints([3, 3, 0, 1, 3, 3, 3, 3])              # rejected drafts
    step(*[1] * 8)
    step(0, 0, 90, 0, 1, 0, 0, 1)                               # more than 16 new tokens a slot in the mean are not needed for this
    step(60, 20, 20, 20, 40, 0, 20, 20)                         # and these are more
    layer.release(1)
    assert layer.kv_len.tolist()[1:4] == [158, 0, 0]
    if own_pages:
        assert torch.equal(layer.table[:5], own[:5])
    else:
        assert layer.table[2:4, :133 // page].eq(-1).all()
        layer.table[2:4] = own[2:4]
    step(1, 1, 50, 2, 1, 1, 1, 1)
    layer.fork(2, 3, 40)
    step(*[1] * 8)
    layer.release(5)
    layer.release(2)
    layer.table.copy_(own)
    step(1, 1, 1, 9, 9, 1, 9, 9)


def test_forked_caches_are_copies():
    """What a fork's slots hold and answer is what they would have held and answered from passes of their own over the prompt."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    rq, rk = ropes(g, 128)
    layer, other = (bx.AttnLayer(4, 200, 4, 2, 128, 16, rope=rq, rope_k=rk, max_forks=1, worth=0) for _ in "ab")
    prompt = drawn(g, 75, 4, 2, 128)
    layer.prefill(ints([0, 75, 75, 75, 75]), 75, *prompt)
    layer.fork(0, 4, 75)
    other.prefill(ints([0, 75, 150, 225, 300]), 75, *(t.repeat(4, 1, 1) for t in prompt))
    for _ in range(30):
        step = drawn(g, 4, 4, 2, 128)
        a, b = layer.decode(*step), other.decode(*step)
        assert (a.double() - b.double()).abs().max() <= 2.0 ** -7 * max(a.abs().max(), 1)
    read = []
    for x in (layer, other):
        n = int(x.kv_len.sum())
        read.append([torch.empty(n, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in "kv"])
        assert bx.ix_kv8_read(x.cache, 4, n, ints(cumulative(x.kv_len.tolist())), x.kv_len, x.table, x.width, *read[-1]) == 0
    assert all(torch.equal(a, b) for a, b in zip(*read))


def test_captured():
    """Replays of a captured token on another stream, while the prompt that is shared and its length change, against eager calls."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(9)
    rq, rk = ropes(g, 64)
    layer, other = (bx.AttnLayer(6, 700, 8, 2, 64, 32, rope=rq, rope_k=rk, max_forks=1, worth=0) for _ in "ab")
    step = drawn(g, 6, 8, 2, 64)
    o = torch.empty_like(step[0])
    graph = torch.cuda.CUDAGraph()
    for tokens in (100, 515, 64):
        prompt = drawn(g, tokens, 8, 2, 64)
        for x in (layer, other):
            if x._forks:
                x.release(1)
            x.kv_len.zero_()
            x.prefill(ints([0, 0] + [tokens] * 5), tokens, *prompt)
            x.fork(1, 5, tokens)
        if tokens == 100:
            held = layer.kv_len.clone()
            with torch.cuda.graph(graph):
                layer.decode(*step, o)
            assert torch.equal(layer.kv_len, held)
        side = torch.cuda.Stream()
        for i in range(8):
            for t in step:
                t.normal_(generator=g)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            side.synchronize()
            assert torch.equal(o, other.decode(*step)), (tokens, i)
        assert layer.kv_len.tolist() == [8] + [tokens + 8] * 5


@pytest.mark.parametrize("as_address", [False, True])
def test_a_stream_that_is_behind(as_address):
    """A prompt, a fork, tokens and a release, all on a stream that is busy when the first is made."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    rq, rk = ropes(g, 64)
    layer, other = (bx.AttnLayer(3, 400, 4, 2, 64, 16, rope=rq, rope_k=rk, max_forks=1, worth=0) for _ in "ab")
    prompt, steps = drawn(g, 301, 4, 2, 64), [drawn(g, 3, 4, 2, 64) for _ in range(4)]
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    cu = ints([0, 301, 301, 301])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 1e-3
    s = side.cuda_stream if as_address else side
    got = [layer.prefill(cu, 301, *prompt, stream=s)]
    behind = not side.query()
    layer.fork(0, 3, 301, stream=s)
    got += [layer.decode(*x, stream=s) for x in steps]
    layer.release(0, stream=s)
    side.synchronize()
    assert behind
    want = [other.prefill(cu, 301, *prompt)]
    other.fork(0, 3, 301)
    want += [other.decode(*x) for x in steps]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert layer.kv_len.tolist() == [305, 0, 0]


def test_refusals():
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    rq, rk = ropes(g, 64)
    with pytest.raises(ValueError):
        bx.AttnLayer(2, 64, 4, 2, 64, 16, rope_k=rk)
    with pytest.raises(ValueError):
        bx.AttnLayer(2, 64, 4, 2, 64, 16, window=8, max_forks=1)
    with pytest.raises(ValueError):
        bx.AttnLayer(2, 64, 4, 2, 64, 16, max_forks=-1)
    layer = bx.AttnLayer(6, 64, 4, 2, 64, 16, rope=rq, rope_k=rk, max_forks=1)
    layer.prefill(ints([0, 20, 20, 40, 40, 40, 40]), 20, *drawn(g, 40, 4, 2, 64))
    table, held = layer.table.clone(), layer.kv_len.clone()
    for bad in ((-1, 2, 20), (0, 1, 20), (5, 2, 20), (0, 7, 20), (0, 2, 0), (0, 2, 21), (0, 2, 65), (1, 2, 1)):
        with pytest.raises(ValueError):
            layer.fork(*bad)
    with pytest.raises(ValueError):
        layer.release(0)
    assert torch.equal(layer.table, table) and torch.equal(layer.kv_len, held)
    layer.fork(0, 2, 20)
    for bad in ((0, 2, 20), (2, 2, 20), (1, 2, 20)):            # a second one
        with pytest.raises(ValueError):
            layer.fork(*bad)
    two = bx.AttnLayer(6, 64, 4, 2, 64, 16, n_pages=10, max_forks=2)
    two.table[:4, :2] = ints([[0, 1], [2, 3], [4, 99], [6, 1]])
    two.prefill(ints([0, 20, 20, 20, 20, 20, 20]), 20, *drawn(g, 20, 4, 2, 64))
    for n in (3, 4, 5):                                         # no place, another slot's, none given
        with pytest.raises(ValueError):
            two.fork(0, n, 20)
    two.fork(0, 2, 20)
    with pytest.raises(ValueError):
        two.fork(1, 3, 20)                                      # a slot of a fork already
    odd = bx.AttnLayer(2, 64, 4, 2, 64, 16, rope=bx.rope(rq.tensors[0], norm=torch.ones(32, device="cuda")))
    with pytest.raises(ValueError):
        odd.decode(*drawn(g, 2, 4, 2, 64))
    far = bx.AttnLayer(2, 64, 4, 2, 64, 16, rope=bx.rope(bx.rope_freq(128)[0].cuda()))
    with pytest.raises(bx.IxGdnError):
        far.decode(*drawn(g, 2, 4, 2, 64))
    assert odd.kv_len.tolist() == far.kv_len.tolist() == [0, 0]


def test_continuations():
    """Continued token by token from one pass over each prompt, the stack ends where a pass over a continuation's tokens ends, within
    what tests/test_attn_layer.py derives for tokens against one prompt."""
    import torch
    from examples import hybrid
    prompts = [[i % 512 for i in range(5, 305)], [1, 2, 3], list(range(64))]
    made, model = hybrid.continuations(prompts, 2, 6)
    assert len(made) == 6 and all(len(m) == 6 for m in made)
    whole = hybrid.Hybrid(6, 400, rope_base=1e4)
    tokens = [prompts[i // 2] + m for i, m in enumerate(made)]
    lens = [len(t) for t in tokens]
    whole.forward(torch.tensor(sum(tokens, []), device="cuda"), ints(cumulative(lens)), max(lens))
    a, b = model.hidden_state.double(), whole.hidden_state.double()
    assert torch.isfinite(a).all()
    assert ((a - b).norm(dim=1) <= 0.125 * b.norm(dim=1)).all(), ((a - b).norm(dim=1) / b.norm(dim=1)).tolist()
