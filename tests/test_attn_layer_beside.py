"""AttnLayers that share their workspaces."""
import pytest

import baloon_amd as bx
from tests.test_attn_layer_fork import drawn
from tests.test_kv8_cache import ints

pytestmark = pytest.mark.gpu


def test_which_are_shared():
    """Those that are large enough; a layer without forks has one, one with forks two."""
    import torch
    a = bx.AttnLayer(8, 300, 8, 2, 128, 16, max_forks=2)
    same = bx.AttnLayer(8, 900, 8, 2, 128, 32, max_forks=2, beside=a)
    assert same._ws is a._ws and same._shared_ws is a._shared_ws
    plain = bx.AttnLayer(8, 300, 8, 2, 128, 16, beside=a)
    assert plain._ws is a._ws and not hasattr(plain, "_shared_ws")
    first = bx.AttnLayer(8, 300, 8, 2, 128, 16, max_forks=1, beside=plain)
    assert first._ws is a._ws and first._shared_ws is not a._shared_ws
    more = bx.AttnLayer(64, 300, 16, 2, 256, 16, max_forks=2, beside=a)
    assert more._shared_ws.numel() > a._shared_ws.numel() and more._ws.numel() > a._ws.numel()
    assert bx.AttnLayer(8, 300, 8, 2, 128, 16, max_forks=2, beside=more)._shared_ws is more._shared_ws
    for wrong in (object(), a._ws, torch.empty(1 << 28, dtype=torch.uint8, device="cuda")):
        with pytest.raises(ValueError):
            bx.AttnLayer(8, 300, 8, 2, 128, 16, beside=wrong)


def test_a_stack_of_them():
    """Three layers of different shapes, called in turn, eagerly and captured, answer bit for bit what layers of their own do."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    shapes = [(8, 2, 256), (8, 4, 64), (4, 2, 128)]
    stack, own, last = [], [], None
    for s in shapes:
        last = bx.AttnLayer(6, 700, *s, 16, max_forks=1, worth=0, beside=last)
        stack.append(last)
        own.append(bx.AttnLayer(6, 700, *s, 16, max_forks=1, worth=0))
    assert len({x._ws.data_ptr() for x in stack}) == len({x._shared_ws.data_ptr() for x in stack}) == 1
    cu = ints([0, 500, 500, 500, 500, 520, 600])
    for a, b, s in zip(stack, own, shapes):
        rows = drawn(g, 600, *s)
        assert torch.equal(a.prefill(cu, 500, *rows), b.prefill(cu, 500, *rows))
        a.fork(0, 4, 500)
        b.fork(0, 4, 500)
    steps = [drawn(g, 6, *s) for s in shapes]
    outs = [torch.empty_like(x[0]) for x in steps]
    for a, b, x in zip(stack, own, steps):
        assert torch.equal(a.decode(*x), b.decode(*x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for a, x, o in zip(stack, steps, outs):
            a.decode(*x, o)
    for i in range(6):
        for x in steps:
            for t in x:
                t.normal_(generator=g)
        graph.replay()
        for a, b, x, o in zip(stack, own, steps, outs):
            assert torch.equal(o, b.decode(*x)), i
            assert torch.equal(a.kv_len, b.kv_len)
