"""Offsets that begin behind the first row, as a part of a larger batch has them: the rows before are neither read nor written."""
import numpy as np
import pytest

import baloon_amd as bx
from tests import kv8_ref
from tests.test_kv8_attn import Problem
from tests.test_kv8_cache import Pair, bf, cumulative, ints


@pytest.mark.gpu
@pytest.mark.parametrize("before", [1, 16, 37, 700])
def test_cache(before):
    import torch
    p = Pair(20, 16, 2, 64, before)
    tables = np.array([[4, 1, 9, 5], [0, 3, 11, 7]], np.int32)
    q, lens = [40, 3], [45, 50]
    bits, x = kv8_ref.normal_bf16(p.g, 43, 2, 2, 64)
    for b, n in enumerate([5, 47]):                             # older tokens
        old, y = kv8_ref.normal_bf16(p.g, n, 2, 2, 64)
        old = bf(old)
        assert bx.ix_kv8_append(p.cache, 1, n, ints([0, n]), ints([n]), ints(tables[b:b + 1]), 4, old[:, 0], old[:, 1]) == 0
        p.ref.append(n, n, tables[b], {"k": y[:, 0], "v": y[:, 1]})
    rows = torch.full((before + 43, 2, 2, 64), 1e30, dtype=torch.bfloat16, device="cuda")
    rows[before:] = bf(bits)
    cu = before + np.array(cumulative(q))
    args = (p.cache, 2, before + 43, ints(cu), ints(lens), ints(tables), 4)
    assert bx.ix_kv8_append(*args, rows[:, 0], rows[:, 1]) == 0
    for b, at in enumerate(cumulative(q)[:-1]):
        p.ref.append(q[b], lens[b], tables[b], {"k": x[at:at + q[b], 0], "v": x[at:at + q[b], 1]})
    p.check(lens, tables)
    out = [torch.full((before + 43, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    assert bx.ix_kv8_read(*args, *out) == 0
    for n, o in zip("kv", out):
        assert bool((o[:before] == 7).all())
        want = np.concatenate([p.ref.tokens(n, lens[b], tables[b])[0][lens[b] - q[b]:] for b in range(2)])
        assert np.all(np.abs(o[before:].float().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("before", [1, 200, 3000])
@pytest.mark.parametrize("lens", [[1, 2, 1], [5, 200, 3], [900, 3, 1100]])
def test_attention(d, before, lens):
    import torch
    P = Problem(lens, [n + 70 * n % 900 for n in lens], 16, 8, d, 2, seed=before)
    P.upload()
    c, n, T, max_q, cu, kv, table, width = P.args()
    q = torch.full((before + T, 16, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    q[before:] = bf(P.q_bits)
    o = torch.full_like(q, 7)
    size = bx.ix_kv8_attn_workspace_size(c, n, before + T, max_q, 16)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    cu = (cu + before).to(torch.int32)
    assert bx.ix_kv8_attn(c, n, before + T, max_q, cu, kv, table, width, q, 16, P.scale, 0, 0, None, o, ws, size) == 0
    assert bool((o[:before] == 7).all())
    P.check(o[before:].float().cpu().numpy())
