"""ix_kv8_attn_workspace_size of a batch does for every smaller one of the same cache and heads."""
import itertools

import pytest

import baloon_amd as bx
from tests.test_kv8_cache import desc

SIZES = [1, 3, 16, 33, 100, 128, 512, 1000, 4096, 10000, 1 << 17, 1 << 20]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,G", [(1, 1), (1, 128), (2, 8), (8, 1), (8, 4), (64, 16), (1024, 2)])
def test_larger_does_for_smaller(d, h, G):
    c = desc(h=h, d=d)
    size = {(T, q): bx.ix_kv8_attn_workspace_size(c, 1, T, q, h * G) for T, q in itertools.product(SIZES, SIZES)}
    for T, q in size:
        assert 0 < size[T, q] <= 81 << 20
        assert bx.ix_kv8_attn_workspace_size(c, 65535, T, q, h * G) == size[T, q]
        assert all(size[t, m] <= size[T, q] for t, m in size if t <= T and m <= q), (T, q)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_workspace_for_prompts_and_pieces(d):
    """Sized for the longest prompt: shorter ones and tokens are taken with it, and are right."""
    import torch
    from tests.test_kv8_attn import Problem
    from tests.test_kv8_cache import bf
    G, h = 8, 2
    n = bx.ix_kv8_attn_workspace_size(desc(h=h, d=d), 1, 40000, 40000, h * G)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")
    for q in (1, 40, 300, 1100):
        P = Problem([q], [q + 500], 16, h, d, G, seed=q)
        P.upload()
        o = torch.empty(q, h * G, d, dtype=torch.bfloat16, device="cuda")
        assert bx.ix_kv8_attn(*P.args(), bf(P.q_bits), h * G, P.scale, 0, 0, None, o, ws, n) == 0, q
        P.check(o.float().cpu().numpy())
