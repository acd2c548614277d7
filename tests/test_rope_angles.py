"""How far an angle of the rotary positions may be off (include/ix_gdn.h): 2^-23 and 2^-51 of itself."""
import os
from fractions import Fraction

import numpy as np
import pytest

import baloon_amd as bx
from tests import kv8_ref
from tests.conftest import ROOT
from tests.test_kv8_cache import bf, cumulative, ints

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")
TURNS = 0.15915494309189535


def off(pos, freq):
    """What the kernels' arithmetic, 64 bits rounded to 32, is off by in radians."""
    turns = float(pos) * float(freq) * TURNS
    turns -= float(np.rint(turns))
    exact = Fraction(pos) * Fraction(float(freq)) / (2 * PI)
    exact -= round(exact)
    d = abs(Fraction(float(np.float32(turns))) - exact)
    return float(min(d, 1 - d) * 2 * PI)


@pytest.mark.parametrize("log", [0, 10, 20, 24, 28, 29, 30])
def test_bound(log):
    g = np.random.default_rng(log)
    worst = 0.0
    for _ in range(4000):
        pos, freq = int(g.integers(1 << log, 2 << log)), np.float32(g.uniform(2.0 ** -20, 1) ** g.choice([0.01, 1, 4]))
        e = off(pos, freq)
        assert e <= 2.0 ** -23 + 2.0 ** -51 * pos * float(freq), (pos, freq)
        worst = max(worst, e)
    assert worst <= (2.0 ** -22 if log < 28 else 2.0 ** -20 + 2.0 ** -23)
    if log == 30:
        assert worst > 2.0 ** -22                               # which is why the bound has a part that grows


def test_the_kernels_compute_it_so():
    text = open(os.path.join(ROOT, "baloon_amd", "csrc", "rope.h")).read()
    assert f"double turns = (double)pos * (double)freq * {TURNS!r};\n    turns -= rint(turns);" in text


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [0, 1])
def test_the_last_positions(layout):
    """Up to 2^31 - 2, against cosines of angles in 80 bits: half a bf16 step (8 bits of a value: 2^-8 of it), the angle, and 2^-20.9 for what 32 bits lose behind
    it (tests/rope_ref.py)."""
    import torch
    g = np.random.default_rng(layout)
    q, kv = [3, 2, 1, 2], [2 ** 31 - 1, (1 << 30) + 7, 1 << 29, 3]
    bits, x = kv8_ref.normal_bf16(g, 8, 4, 128)
    freq = np.concatenate([[1.0], g.uniform(0.5, 1, 31), 1e4 ** (-np.arange(32) / 32)]).astype(np.float32)
    y = torch.empty(8, 4, 128, dtype=torch.bfloat16, device="cuda")
    r = bx.rope(torch.from_numpy(freq).cuda(), layout)
    assert bx.ix_rope_rows(r, 4, 8, ints(cumulative(q)), ints(kv), bf(bits), 4, 128, y) == 0
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(q, kv)])
    angle = pos[:, None, None].astype(np.longdouble) * freq.astype(np.longdouble)
    assert np.finfo(angle.dtype).nmant >= 63
    c, s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    i = np.arange(64)
    a, b = (2 * i, 2 * i + 1) if layout else (i, i + 64)
    want, e = x.astype(np.float64), np.zeros(x.shape)
    want[..., a], want[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    e[..., a] = e[..., b] = (2.0 ** -23 + 2.0 ** -51 * angle.astype(np.float64) + 2.0 ** -20.9) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    got = y.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 1.01 * e)
