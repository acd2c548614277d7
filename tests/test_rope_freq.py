"""baloon_amd.rope_freq's two scalings by parts, each against numbers worked out by hand from its own definition."""
import math

import pytest

import baloon_amd as bx


def kept(freq, base, rot, factor):
    """How much of each frequency is kept: 1 whole, 0 divided by factor."""
    return [(float(f) * base ** (2 * i / rot) - 1 / factor) / (1 - 1 / factor) for i, f in enumerate(freq)]


def test_by_channels():
    """rot 128, base 10,000, 4,096 tokens: pair i goes round 4096 / 2 pi * 10000 ** (-i / 64) = 651.899 e^(-0.14391 i) times: 32 at
    i = 20.94 and once at 45.03. So the pairs up to 20 are kept, those from 46 on divided, and pair i between keeps (46 - i) / 26."""
    freq, amplitude = bx.rope_freq(128, 1e4, "channels", 4.0, trained=4096)
    assert math.isclose(amplitude, 0.1 * math.log(4) + 1)
    for i, k in enumerate(kept(freq, 1e4, 128, 4.0)):
        assert abs(k - min(max((46 - i) / 26, 0), 1)) < 2.0 ** -20, i


def test_by_parts():
    """The same by rounds: pair i keeps (rounds - 1) / 31."""
    freq, amplitude = bx.rope_freq(128, 1e4, "parts", 4.0, trained=4096)
    assert math.isclose(amplitude, 0.1 * math.log(4) + 1)
    for i, k in enumerate(kept(freq, 1e4, 128, 4.0)):
        assert abs(k - min(max((4096 / (2 * math.pi) * 1e4 ** (-i / 64) - 1) / 31, 0), 1)) < 2.0 ** -20, i


def test_how_far_they_differ():
    a, b = (bx.rope_freq(64, 1e7, s, 4.0, trained=262144)[0] for s in ("parts", "channels"))
    off = (a / b - 1).abs()
    assert int((off > 1e-6).sum()) == 7 and 0.45 < float(off.max()) < 0.46


@pytest.mark.parametrize("slow,fast,lo,hi", [(1.0, 32.0, 1, 5), (1.0, 1e6, 0, 5), (0.001, 0.002, 9, 11)])
def test_limits_outside_the_pairs(slow, fast, lo, hi):
    """rot 16, base 10,000, 1,000 tokens: 159.15 e^(-1.15129 i) rounds. 32 at 1.39, 1 at 4.40; 0.002 at 9.80, 0.001 at 10.41: beyond the
    last pair, 7, so all are kept; 1e6 before the first."""
    k = kept(bx.rope_freq(16, 1e4, "channels", 8.0, trained=1000, slow=slow, fast=fast)[0], 1e4, 16, 8.0)
    for i, x in enumerate(k):
        assert abs(x - min(max((hi - i) / (hi - lo), 0), 1)) < 2.0 ** -20, i


def test_refusals():
    for kw in (dict(trained=None), dict(trained=0), dict(trained=-5), dict(trained=4096, slow=0.0), dict(trained=4096, slow=4.0, fast=4.0)):
        with pytest.raises(ValueError):
            bx.rope_freq(64, 1e4, "channels", 2.0, **kw)
