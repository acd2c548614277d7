"""Shared tokens beyond position 2^30: pages that a table names again and again stand for them."""
import numpy as np
import pytest

import baloon_amd as bx
from tests.test_kv8_cache import cumulative, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40])
def test_shared_tokens_far_on(new):
    """2^30 + 4,224 shared tokens of which those of page 1, the last 4,096 whole ones and so far on, weigh e^40 times as much as the others (page 0):
    the output is the mean of page 1's values, less 2^30 / (4,096 e^40) < 2^-40 of it. q is exact in its 16 bits, the score 40 is within
    2^-20 of itself the same for all of page 1, P's rounding to fp16 2^-11 of the largest value, the result's
    to bf16, of 8 bits, 2^-8 of it."""
    import torch
    g = np.random.default_rng(new)
    page, d, far = 128, 64, 2 ** 30 + 128
    shared = far + 4096
    pages = shared // page
    width = pages + 1
    k, v = np.zeros((4, 1, page, d), np.int8), np.zeros((4, 1, d, page), np.int8)
    k[1] = 100
    v[1] = g.integers(-127, 128, (1, d, page))
    scale = np.full((4, 1), 0.01, np.float32)
    cache = bx.kv8_cache(*(torch.from_numpy(x).cuda() for x in (k, v, scale, scale)))
    table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    table[:, far // page:pages] = 1
    table[:, pages] = ints([2, 3])
    q = torch.full((2 * new, 1, d), 1.0, dtype=torch.bfloat16, device="cuda")
    o = torch.full_like(q, float("nan"))
    a = (cache, 2, 2 * new, new, ints(cumulative([new, new])), ints([shared + new] * 2), table, width, 1, ints([0, 2]), ints([shared]), q, 1, 40 / 64, None, o)
    n = bx.ix_kv8_attn_shared_workspace_size(cache, 2, 2 * new, new, 1, 1)
    assert bx.ix_kv8_attn_shared(*a, torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda"), n) == 0
    want = v[1, 0].astype(np.float64).mean(1) * np.float64(np.float32(0.01))
    got = o.double().cpu().numpy()
    off = 2.0 ** -8 * np.abs(want) + 2.0 ** -11 * 1.27
    assert np.all(np.abs(got - want) <= off), (got[0, 0, :5], want[:5])
