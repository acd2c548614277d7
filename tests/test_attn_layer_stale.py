"""Captured calls of an AttnLayer whose forks change afterwards."""
import pytest

import baloon_amd as bx
from tests.test_attn_layer_fork import drawn
from tests.test_kv8_cache import ints

pytestmark = pytest.mark.gpu


def captured(layer, step):
    import torch
    o, held, graph = torch.empty_like(step[0]), layer.kv_len.clone(), torch.cuda.CUDAGraph()
    layer.decode(*step, o)                                      # and back, so that what a first call sets up is not captured
    layer.kv_len.copy_(held)
    with torch.cuda.graph(graph):
        layer.decode(*step, o)
    assert torch.equal(layer.kv_len, held)
    return graph, o


def prompt(layer, g, lens):
    layer.kv_len.zero_()
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return layer.prefill(ints(cu), max(lens), *drawn(g, cu[-1], layer.h_q, layer.h_kv, layer.d))


@pytest.mark.parametrize("d", [64, 256])
def test_forks_that_change(d):
    """Graphs of a token, made with two forks, with one and with none, replayed after forks were made and released: each time what a
    layer without forks answers from the same pages. 2^-7 of the largest output: two results of one's tolerance each."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(d)
    layer = bx.AttnLayer(9, 600, 8, 2, d, 16, max_forks=2, worth=0)
    step = drawn(g, 9, 8, 2, d)
    alone = bx.AttnLayer(9, 600, 8, 2, d, 16)
    graphs = {}

    def check(what):
        for name, (graph, o) in graphs.items():
            for t in step:
                t.normal_(generator=g)
            for a, b in zip(alone.cache.tensors, layer.cache.tensors):
                a.copy_(b)
            alone.table.copy_(layer.table)
            alone.kv_len.copy_(layer.kv_len)
            o.fill_(7.0)
            graph.replay()
            want = alone.decode(*step)
            torch.cuda.synchronize()
            assert (o.double() - want.double()).abs().max() <= 2.0 ** -7 * max(float(want.abs().max()), 1), (what, name)
            assert torch.equal(layer.kv_len, alone.kv_len)

    graphs["none"] = captured(layer, step)
    prompt(layer, g, [300, 20, 5, 77, 8, 200, 9, 9, 9])
    check("before")
    layer.fork(0, 3, 300)
    graphs["one"] = captured(layer, step)
    layer.fork(5, 4, 200)
    graphs["two"] = captured(layer, step)
    check("two forks")
    layer.release(0)
    check("the first released")
    layer.release(5)
    prompt(layer, g, [30, 20, 5, 400, 8, 210, 40, 41, 250])
    check("none")
    layer.fork(3, 2, 400)
    check("another")
    layer.release(3)
    prompt(layer, g, [250, 240, 230, 220, 210, 200, 190, 180, 170])
    check("none again")
