"""More workgroups than a launch can have (2^32 threads a dimension): rows of the norm, room for tokens in the cache's calls,
blocks of rows in the attention."""
import numpy as np
import pytest

import baloon_amd as bx
from tests import kv8_ref
from tests.test_kv8_cache import Pair, bf, ints

INVALID = bx.HIP_ERROR_INVALID_VALUE
A = 1 << 20


def test_refusals():
    """Room for so many rows that blocks of them could not be numbered."""
    from tests.test_kv8_attn import attn, desc
    assert attn(desc(h=1), T=2 ** 31 - 1, max_q=2 ** 31 - 1, h_q=4096, q=(A, 4096 * 64)) == INVALID


@pytest.mark.gpu
def test_norm_rows():
    """Rows of 32 in a pattern: each equals its small call's."""
    import torch
    m, n = 1024, 32
    rows = (1 << 26) + 5                                       # a workgroup of 64 threads each
    g = np.random.default_rng(1)
    part = bf(kv8_ref.normal_bf16(g, m, n)[0])
    w = torch.linspace(0.5, 2, n, device="cuda")

    def call(x):
        h, y16 = torch.empty_like(x), torch.empty_like(x)
        y = torch.empty(x.shape, device="cuda")
        q = torch.empty(x.shape[0], 36, dtype=torch.uint8, device="cuda")
        assert bx.ix_add_rms_norm(x.shape[0], n, x, x, h, w, 0.0, 1e-6, y, y16, q) == 0
        return h, y, y16, q

    want = call(part)
    got = call(part.repeat(rows // m + 1, 1)[:rows])
    for a, b in zip(got, want):
        whole = rows // m * m
        assert torch.equal(a[whole:], b[:rows - whole])
        for i in range(0, whole, m << 12):
            c = a[i:i + (m << 12)].view(-1, *b.shape)
            assert bool((c == b).all()), i


@pytest.mark.gpu
def test_room_for_tokens():
    """The offsets use 3 + 120 of 2^29 rows."""
    import torch
    p = Pair(12, 16, 1, 256, 5)
    T = 1 << 29
    tables = np.array([[4, -1, -1, -1, -1, -1, -1, -1], [0, 3, 9, 11, 2, 1, 7, 8]], np.int32)
    bits, x = kv8_ref.normal_bf16(p.g, 123, 2, 1, 256)
    rows = bf(bits)
    p.ref.append(3, 3, tables[0], {"k": x[:3, 0], "v": x[:3, 1]})
    p.ref.append(120, 120, tables[1], {"k": x[3:, 0], "v": x[3:, 1]})
    args = (p.cache, 2, T, ints([0, 3, 123]), ints([3, 120]), ints(tables), 8)
    assert bx.ix_kv8_append(*args, rows[:, 0], rows[:, 1]) == 0
    p.check([3, 120], tables)
    out = [torch.full((123, 1, 256), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    assert bx.ix_kv8_read(*args, *out) == 0
    for n, o in zip("kv", out):
        want = np.concatenate([p.ref.tokens(n, 3, tables[0])[0], p.ref.tokens(n, 120, tables[1])[0]])
        err = np.abs(o.float().cpu().numpy() - want)
        assert np.all(err <= 2.0 ** -8 * np.abs(want))


@pytest.mark.gpu
def test_attention_of_many_sequences_and_heads():
    """65,535 sequences, nearly all without a new token, and 256 heads. Tolerance: tests/test_kv8_attn.py's with its terms at these
    sizes: scores under 64 of which q's 16 bits and 32-bit sums move 2^-11, and 2^-11 for p, twice."""
    import torch
    n, h, d = 65535, 256, 64
    q, kv = np.zeros(n, np.int64), np.zeros(n, np.int64)
    some = {0: (100, 150), 300: (60, 60), 40000: (5, 33), n - 1: (120, 121)}
    tables, page = np.full((n, 10), -1, np.int32), 0
    for b, (m, k) in some.items():
        q[b], kv[b] = m, k
        tables[b, :-(-k // 16)] = np.arange(page, page + -(-k // 16))
        page += -(-k // 16)
    p = Pair(page, 16, h, d, 3)
    for s in "kv":
        p.ref.codes[s][:] = np.clip(np.rint(p.g.normal(0, 40, p.ref.codes[s].shape)), -127, 127).astype(np.int8)
        p.ref.scale[s][:] = (p.g.uniform(0.5, 1.5, p.ref.scale[s].shape) / 40).astype(np.float32)
    c, s, t = p.ref.codes, p.ref.scale, p.t
    for at, x in zip(t, (c["k"], np.ascontiguousarray(c["v"].swapaxes(2, 3)), s["k"], s["v"])):
        at.copy_(torch.from_numpy(x.copy()))
    T = int(q.sum())
    bits, qv = kv8_ref.normal_bf16(p.g, T, h, d)
    o = torch.full((T, h, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    size = bx.ix_kv8_attn_workspace_size(p.cache, n, T, 120, h)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    assert bx.ix_kv8_attn(p.cache, n, T, 120, ints(np.concatenate([[0], np.cumsum(q)])), ints(kv), ints(tables), 10, bf(bits), h, d ** -0.5,
                          0, 0, None, o, ws, size) == 0
    got, at = o.float().cpu().numpy(), 0
    for b, (m, k) in some.items():
        (kk, has), (vv, _) = p.ref.tokens("k", k, tables[b]), p.ref.tokens("v", k, tables[b])
        want = kv8_ref.attend(qv[at:at + m], k, kk, vv, kv8_ref.seen_by(m, k, has, 0, 0), d ** -0.5)
        assert np.all(np.abs(got[at:at + m] - want) <= np.abs(vv).max() * 2.0 ** -9 + 2.0 ** -8 * np.abs(want)), b
        at += m
