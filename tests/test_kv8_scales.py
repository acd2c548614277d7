"""ix_kv8_attn over pages of any scales: what lies in memory that no sequence uses, pages of values next to nothing, pages whose
scales are far apart. A page's value scale weighs its values; the softmax's sum does not know it.

Tolerance: that of tests/test_kv8_attn.py, of which nothing depends on the scales (the values' product holds p vs in fp16
relative to the largest, 2^-33 of it or 2^-11 of its own: both relative to max|v|), and 2^-126, the smallest normal number,
below which results may be flushed."""
import numpy as np
import pytest

from oracle import bf16
from tests import kv8_ref
from tests.test_kv8_attn import Problem
from tests.test_kv8_cache import cumulative

F = np.float32
# bits of integers of another use, subnormal and small numbers, and what 1 / x of is infinite
LEFT = [F(1e-45), F(1e-40), F(2.0 ** -128), F(2.0 ** -127), np.array([(1 << 21) - 1], np.int32).view(F)[0],
        F(1e-37), F(3e38), F(-1e-40), F(np.nan), F(np.inf), F(0)]


def check(P, got, window=0, sinks=0, scale=None):
    """Problem.check, results below 2^-126 aside."""
    scale = P.scale if scale is None else scale
    at = 0
    for b, (m, n) in enumerate(zip(P.q_len, P.kv_len)):
        k, has = P.p.ref.tokens("k", n, P.tables[b])
        v, _ = P.p.ref.tokens("v", n, P.tables[b])
        seen = kv8_ref.seen_by(m, n, has, window, sinks)
        k[~seen.any(0)] = 0
        v[~seen.any(0)] = 0
        q = P.q[at:at + m]
        want = kv8_ref.attend(q, n, k, v, seen, scale)
        amax, sum_k = np.abs(q).max(2, keepdims=True), np.abs(k).sum(2).max()
        e1 = abs(scale) * amax / 65278 * sum_k
        e2 = 2.0 ** -22 * (abs(scale) * amax * sum_k + 16) * 1.5
        tol = np.abs(v).max() * (2 * (e1 + e2) + 2.0 ** -11 + n * 2.0 ** -32 + (n / 16 + 64) * 2.0 ** -23) + 2.0 ** -8 * np.abs(want) + 2.0 ** -126
        near = np.abs(got[at:at + m] - want) <= tol
        assert near.all(), (b, np.argwhere(~near)[:5], got[at:at + m][~near][:5], want[~near][:5], tol[~near][:5])
        at += m


def free_page_0(P):
    """Page 0 and at least 7 others belong to no sequence; all of them hold the codes and scales `LEFT`."""
    used = set(P.tables[P.tables >= 0].tolist())
    other = sorted(set(range(P.p.ref.n_pages)) - used)
    if 0 in used:
        P.tables[P.tables == 0] = other[-1]
        other[-1] = 0
    return sorted(other)


# (new tokens, sequences, heads): a token and drafts by the wave, blocks of rows, and those in parts
SHAPES = [(1, 3, 2), (3, 3, 2), (500, 2, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,n,h", SHAPES)
@pytest.mark.parametrize("left", range(len(LEFT)))
def test_scales_of_pages_that_nobody_has(d, q, n, h, left):
    """Whatever page 0 and the others hold: pages end inside a tile, a sequence has pages that are gone."""
    P = Problem([q] * n, [q + 203 * b + 9 for b in range(n)], 16, h, d, 4, seed=left, spare=8)
    for i in free_page_0(P):
        for s in "kv":
            P.p.ref.codes[s][i] = -128
            P.p.ref.scale[s][i] = LEFT[left]
    P.tables[n - 1, 3] = -1
    P.both()
    P.both(window=70, sinks=5)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,n,h", SHAPES)
@pytest.mark.parametrize("tiny", [2.0 ** -149, 2.0 ** -140, 2.0 ** -128, 2.0 ** -126, 2.0 ** -100])
def test_pages_of_values_next_to_nothing(d, q, n, h, tiny):
    """Partly filled, hidden from some rows and seen by others; then the whole cache, whose results are themselves that small."""
    P = Problem([q] * n, [q + 203 * b + 9 for b in range(n)], 16, h, d, 4, seed=int(-np.log2(tiny)))
    ref = P.p.ref
    for b in range(n):
        last = (P.kv_len[b] - 1) // 16
        for p in {0, last // 2, last}:
            ref.scale["v"][P.tables[b, p]] = F(tiny)
    check(P, P.run())
    check(P, P.run(window=70, sinks=5), window=70, sinks=5)
    ref.scale["v"][:] = F(tiny)
    check(P, P.run())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,n,h", SHAPES)
@pytest.mark.parametrize("apart", [20, 24, 26, 28, 30, 34, 40, 60, 100, 140, None])
@pytest.mark.parametrize("flat", [True, False])
def test_pages_far_apart(d, q, n, h, apart, flat):
    """Every other page's values are 2^-apart of the others' (0 for None): with equal scores their tokens hold half of the weight,
    with scores of the usual spread theirs is as good."""
    P = Problem([q] * n, [q + 203 * b + 9 for b in range(n)], 16, h, d, 4, seed=d + q, q_std=0.0 if flat else 1.0)
    ref = P.p.ref
    big = 2.0 ** 20 if apart == 140 else 1.0
    ref.scale["v"][:] *= F(big)
    for b in range(n):
        for p in range(b % 2, -(-P.kv_len[b] // 16), 2):
            if apart is None:
                ref.codes["v"][P.tables[b, p]] = 0
                ref.scale["v"][P.tables[b, p]] = 0
            else:
                ref.scale["v"][P.tables[b, p]] *= F(2.0 ** -apart)
    check(P, P.run())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,n,h", SHAPES)
@pytest.mark.parametrize("small", [1e-8, 1e-10, 1e-12, 1e-20, 1e-30])
def test_pages_of_zeros_beside_small_ones(d, q, n, h, small):
    P = Problem([q] * n, [q + 203 * b + 9 for b in range(n)], 16, h, d, 4, seed=3, v_std=small)
    for b in range(n):
        for p in range(1 - b % 2, -(-P.kv_len[b] // 16), 3):
            P.p.ref.codes["v"][P.tables[b, p]] = 0
            P.p.ref.scale["v"][P.tables[b, p]] = 0
    check(P, P.run())


@pytest.mark.gpu
@pytest.mark.parametrize("q,n,h", SHAPES)
@pytest.mark.parametrize("d", [64, 256])
def test_weight_on_small_values(d, q, n, h):
    """The tokens that hold nearly all of the weight are of a page of values 2^-40 of the others'; the others' weights, 2^-40 too,
    make half of the result."""
    P = Problem([q] * n, [q + 203 * b + 9 for b in range(n)], 16, h, d, 4, seed=5)
    ref = P.p.ref
    P.q[:] = 0
    P.q[:, :, 0] = 8
    P.q_bits = bf16.from_f32(P.q)
    ref.scale["k"][:] = F(1 / 127)
    ref.codes["k"][:] = 0
    for b in range(n):
        first = P.tables[b, 0]
        ref.codes["k"][first, :, :, 0] = 127
        ref.scale["v"][first] *= F(2.0 ** -40)
    ref.codes["v"][:] = np.abs(ref.codes["v"])
    scale = float(40 * np.log(2) / 8)
    got = P.run(scale=scale)
    # the results are 2^-40 of max|v|: relative to them, by the definition's error for p (2^-10 of each term, all of one sign)
    at = 0
    for b, (m, kv) in enumerate(zip(P.q_len, P.kv_len)):
        k, has = ref.tokens("k", kv, P.tables[b])
        v, _ = ref.tokens("v", kv, P.tables[b])
        seen = kv8_ref.seen_by(m, kv, has, 0, 0)
        want = kv8_ref.attend(P.q[at:at + m], kv, k, v, seen, scale)
        # scores: e1 and e2 of the module's tolerance at 40 ln 2 (each term moves by them), fp16's 2^-11, the result's 2^-8
        sum_k = np.abs(k).sum(2).max()
        rel = 2 * (scale * 8 / 65278 * sum_k + 2.0 ** -22 * (scale * 8 * sum_k + 16) * 1.5) + 2.0 ** -10 + 2.0 ** -8
        assert np.all(np.abs(got[at:at + m] - want) <= rel * np.abs(want)), np.abs(got[at:at + m] / want - 1).max()
        at += m


@pytest.mark.gpu
def test_rows_keep_their_bits_beside_others():
    """A row's result is its own: the same bits with rows beside it whose scores are not finite or far larger, over pages far apart."""
    for q in (3, 130, 600):
        P = Problem([q, q], [q + 70, q + 9], 16, 2, 128, 8, seed=q)
        for p in range(0, P.p.ref.n_pages, 2):
            P.p.ref.scale["v"][p] *= F(2.0 ** -70)
        clean = P.run()
        P.q[0, 3] = np.nan
        P.q[1, 15, 7] = np.inf
        P.q_bits = bf16.from_f32(P.q)
        got = P.run()
        for t, hh in ((0, 3), (1, 15)):
            got[t, hh] = clean[t, hh]
        assert np.array_equal(got, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,n,h", SHAPES)
@pytest.mark.parametrize("first,others", [(3e4, 0), (0, -3e4), (-1e6, -2e6), (1e6, -1e6), (2e7, 1e7)])
def test_one_token_far_above_the_others(d, q, n, h, first, others):
    """Scores far from 0 of which the first token's is so much larger that it has all of the weight: the result is its value, and the
    scores' size is no part of the tolerance (2^-11 for p in fp16 and 2^-8 for the result's half ulp, as in the module's)."""
    P = Problem([q] * n, [q + 203 * b + 9 for b in range(n)], 16, h, d, 4, seed=7)
    ref = P.p.ref
    P.q[:] = 0
    P.q[:, :, 0] = 8
    P.q_bits = bf16.from_f32(P.q)
    unit = 1e4 if max(abs(first), abs(others)) < 1e6 else 1e6
    ref.codes["k"][:] = 0
    ref.codes["k"][:, :, :, 0] = int(others / unit)
    for b in range(n):
        ref.codes["k"][P.tables[b, 0], :, 0, 0] = int(first / unit)
    ref.scale["k"][:] = 1
    got, at = P.run(scale=unit / 8), 0
    for b, m in enumerate(P.q_len):
        v, _ = ref.tokens("v", 1, P.tables[b])
        want = v[0].astype(np.float64).repeat(4, 0)[None]
        assert np.all(np.abs(got[at:at + m] - want) <= (2.0 ** -11 + 2.0 ** -8) * np.abs(want) + 2.0 ** -33 * np.abs(v).max())
        at += m
