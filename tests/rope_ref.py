"""A head's rotary positions and norm in plain numpy, in 64 bits, from their definition (include/ix_gdn.h)."""
import numpy as np


def turned(x, pos, freq, pairs=False, amplitude=1.0, norm=None, offset=0.0, eps=1e-6):
    """x [T][heads][d], pos [T] -> (y, what a 32-bit form may be off by before its rounding to bf16).

    Errors of a 32-bit form: an angle by 2^-23.3 (half a turn rounded to 32 bits, in radians) + 2^-22 (a position of 30 bits times a
    frequency, in 64), cos and sin by 2^-23 and their product with the amplitude 2^-24, products and sum 3 2^-24: under 2^-20.9 of
    amplitude (|f_a| + |f_b|). A norm: the sum of squares by at most 20 roundings of 2^-24 / 2, its root's reciprocal 2^-23, two
    products 2^-23: under 2^-20.2 of f. 2^-19.4 of both, and nothing for a channel that passes without a norm."""
    f = x.astype(np.float64)
    d, rot = x.shape[2], 2 * len(freq)
    if norm is not None:
        f = f / np.sqrt((f * f).mean(2, keepdims=True) + eps) * (np.float64(offset) + norm.astype(np.float64))
    angle = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freq, np.float64)
    c, s = amplitude * np.cos(angle), amplitude * np.sin(angle)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if pairs else (i, i + rot // 2)
    y = f.copy()
    y[..., a] = f[..., a] * c - f[..., b] * s
    y[..., b] = f[..., b] * c + f[..., a] * s
    off = 2.0 ** -20.2 * np.abs(f) if norm is not None else np.zeros_like(f)
    off[..., a] = off[..., b] = 2.0 ** -19.4 * abs(amplitude) * (np.abs(f[..., a]) + np.abs(f[..., b]))
    return y, off
