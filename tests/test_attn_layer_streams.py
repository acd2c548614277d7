"""AttnLayer on another stream than torch's current one, and captured: a call's lengths, kernels and outputs are in its stream's order,
and its workspace stays where it is."""
import ctypes

import pytest

import baloon_amd as bx
from tests.test_attn_layer_calls import rows
from tests.test_kv8_cache import ints

pytestmark = pytest.mark.gpu
N, H_Q, H_KV = 3, 4, 2


def layers(n=2, **kw):
    return [bx.AttnLayer(N, 4000, H_Q, H_KV, 64, 16, **kw) for _ in range(n)]


def steps(g):
    """(offsets, longest, q, k, v, gate) of a prompt, tokens and drafts."""
    out = []
    for lens in ((37, 5, 200), (1, 1, 1), (1, 1, 1), (4, 0, 4), (1, 1, 1)):
        T = sum(lens)
        out.append((ints([0, lens[0], lens[0] + lens[1], T]), max(lens), *(rows(g, T, h) for h in (H_Q, H_KV, H_KV, H_Q))))
    return out


def call(layer, step, **kw):
    cu, longest, q, k, v, z = step
    return layer.decode(q, k, v, z, **kw) if q.shape[0] == N else layer.prefill(cu, longest, q, k, v, z, **kw)


@pytest.mark.parametrize("as_address", [False, True])
@pytest.mark.parametrize("own_o", [False, True])
def test_a_stream_that_is_behind(as_address, own_o):
    """All calls are made while the stream is busy with something else: none has begun when the last is made."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    layer, other = layers()
    todo = steps(g)
    want = [call(other, s) for s in todo]
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    o = [torch.empty_like(w) if own_o else None for w in want]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 1e-3
    got = [call(layer, s, o=x, stream=side.cuda_stream if as_address else side) for s, x in zip(todo, o)]
    behind = not side.query()
    side.synchronize()
    assert behind
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert layer.kv_len.tolist() == other.kv_len.tolist() == [44, 8, 207]


@pytest.mark.parametrize("null", [0, "c_void_p", "default"])
def test_the_null_stream_by_its_address(null):
    """While torch's current stream is another one and the null stream is busy."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    layer, other = layers()
    todo = steps(g)
    want = [call(other, s) for s in todo]
    side, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    default = torch.cuda.default_stream()
    torch.cuda.synchronize()
    for _ in range(20):
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(side):
        stream = {0: 0, "c_void_p": ctypes.c_void_p(0), "default": default}[null]
        got = [call(layer, s, stream=stream) for s in todo]
    side_done, behind = side.query(), not default.query()
    torch.cuda.synchronize()
    assert side_done and behind
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_streams_in_turn():
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    layer, other = layers()
    todo = steps(g)
    want = [call(other, s) for s in todo]
    side = torch.cuda.Stream()
    got = []
    for i, s in enumerate(todo):
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
            got.append(call(layer, s, stream=side))
            torch.cuda.current_stream().wait_stream(side)
        else:
            got.append(call(layer, s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_tokens_around_a_long_prompt():
    """A captured decode() replays right after the layer has taken a larger batch than any before the capture."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    layer, other = layers()
    first, token = steps(g)[:2]
    T = 3 * 1200
    prompt = (ints([0, 1200, 2400, T]), 1200, *(rows(g, T, h) for h in (H_Q, H_KV, H_KV, H_Q)))
    for x in (layer, other):
        call(x, first)
    q, k, v, z = (t.clone() for t in token[2:])
    o, lens = torch.empty_like(q), layer.kv_len.clone()
    where = layer._ws.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(layer, (None, 1, q, k, v, z), o=o, stream=side)      # as torch asks: once before the capture
    torch.cuda.current_stream().wait_stream(side)
    layer.kv_len.copy_(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(layer, (None, 1, q, k, v, z), o=o)
    assert layer.kv_len.tolist() == lens.tolist()

    def replay():
        graph.replay()
        want = call(other, (None, 1, q, k, v, z))
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        assert layer.kv_len.tolist() == other.kv_len.tolist()

    replay()
    replay()
    assert torch.equal(call(layer, prompt), call(other, prompt))
    assert layer._ws.data_ptr() == where
    taken = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(100)]      # whatever memory was free
    for _ in range(3):
        replay()
    assert all(bool(t.isnan().all()) for t in taken)
