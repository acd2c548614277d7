"""AttnLayer's calls that raise: the lengths and the cache stay as they were, and the next call's result is as if there had been
none."""
import ctypes

import pytest

import baloon_amd as bx
from tests.test_kv8_cache import ints

pytestmark = pytest.mark.gpu


def rows(g, T, h, d=64):
    import torch
    return torch.randn(T, h, d, generator=g, device="cuda").bfloat16()


def test_calls_that_raise():
    import torch
    n, h_q, h_kv = 2, 4, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    layer, other = (bx.AttnLayer(n, 64, h_q, h_kv, 64, 16) for _ in "ab")
    first = [rows(g, 7, h) for h in (h_q, h_kv, h_kv)]
    for x in (layer, other):
        x.prefill(ints([0, 3, 7]), 4, *first)
    q, k, v, z = (rows(g, 2, h) for h in (h_q, h_kv, h_kv, h_q))
    k *= 10                                                    # a page's scale would grow
    o = torch.empty(2, h_q, 64, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(2, h_q, 128, dtype=torch.bfloat16, device="cuda")
    cu, before = ints([0, 1, 2]), [t.clone() for t in layer.cache.tensors]
    bad = {
        "fp32 q": lambda: layer.decode(q.float(), k, v),
        "fp16 q": lambda: layer.decode(q.half(), k, v),
        "fp32 k": lambda: layer.decode(q, k.float(), v),
        "fp32 v": lambda: layer.decode(q, k, v.float()),
        "fp32 gate": lambda: layer.decode(q, k, v, z.float()),
        "gate on the CPU": lambda: layer.decode(q, k, v, z.cpu()),
        "k on the CPU": lambda: layer.decode(q, k.cpu(), v),
        "rows not dense": lambda: layer.decode(wide[:, :, :64], k, v),
        "gate not dense": lambda: layer.decode(q, k, v, wide[:, :, ::2]),
        "heads and channels turned": lambda: layer.decode(q, k.transpose(1, 2), v),
        "too few heads": lambda: layer.decode(q[:, :2], k, v),
        "too few channels": lambda: layer.decode(q, k[:, :, :32].contiguous(), v),
        "one row for all": lambda: layer.decode(q[:1].expand(2, h_q, 64), k, v),
        "flat q": lambda: layer.decode(q.view(-1)[:2], k, v),
        "o fp32": lambda: layer.decode(q, k, v, None, o.float()),
        "o too small": lambda: layer.decode(q, k, v, None, o[:1]),
        "o not contiguous": lambda: layer.decode(q, k, v, None, wide[:, :, :64]),
        "o on the CPU": lambda: layer.decode(q, k, v, None, o.cpu()),
        "offsets of 64 bits": lambda: layer.prefill(cu.long(), 1, q, k, v),
        "offsets on the CPU": lambda: layer.prefill(cu.cpu(), 1, q, k, v),
        "no tokens at most": lambda: layer.prefill(cu, 0, q, k, v),
        "max_q no number": lambda: layer.prefill(cu, "1", q, k, v),
    }
    for name, call in bad.items():
        with pytest.raises((ValueError, TypeError, AttributeError, ctypes.ArgumentError, bx.IxGdnError)):
            call()
        assert layer.kv_len.tolist() == [3, 4], name
        for a, b in zip(before, layer.cache.tensors):
            assert torch.equal(a, b), name
    got, want = (x.decode(q, k, v, z) for x in (layer, other))
    assert torch.equal(got, want) and layer.kv_len.tolist() == [4, 5]


def test_wider_rows_and_outputs():
    """What was taken is still: rows that go on behind their heads, and a larger o."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    layer, other = (bx.AttnLayer(1, 64, 4, 2, 64, 16) for _ in "ab")
    q, k, v = rows(g, 5, 6), rows(g, 5, 3), rows(g, 5, 3)
    o = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert layer.prefill(ints([0, 5]), 5, q, k, v, None, o) is o
    want = other.prefill(ints([0, 5]), 5, q[:, :4].contiguous(), k[:, :2].contiguous(), v[:, :2].contiguous())
    assert torch.equal(o[:5], want)
