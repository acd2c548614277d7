"""The 8-bit cache and the attention over it in plain numpy, from their definitions (include/ix_gdn.h): codes and
scales in IEEE fp32 as the cache defines them bit for bit, attention in 64 bits."""
import numpy as np

from oracle import bf16

F = np.float32


class Cache:
    """Codes token by token for both (the library's values lie channel by channel), and tables of pages."""

    def __init__(self, n_pages, page, h, d, g):
        self.n_pages, self.page, self.h, self.d = n_pages, page, h, d
        # whatever the memory held before: codes of any value, scales that are not numbers
        self.codes = {n: g.integers(-128, 128, (n_pages, h, page, d)).astype(np.int8) for n in "kv"}
        self.scale = {n: np.full((n_pages, h), np.nan, F) for n in "kv"}

    def place(self, table, p):
        i = table[p] if p < len(table) else -1
        return i if 0 <= i < self.n_pages else None

    def append(self, q, kv_len, table, rows):
        """rows: {"k": [q][h][d] fp32 (bf16 values), "v": ...} of one sequence."""
        first = kv_len - q
        start = max(first, 0)
        for p in range(start // self.page, (kv_len - 1) // self.page + 1 if q and kv_len > 0 else 0):
            at = self.place(table, p)
            lo, hi = max(start, p * self.page), min(kv_len, (p + 1) * self.page)
            if at is None or hi <= lo:
                continue
            held = lo - p * self.page
            for n in "kv":
                x = rows[n][lo - first:hi - first].transpose(1, 0, 2)                      # [h][new][d]
                old = self.scale[n][at] if held else np.zeros(self.h, F)
                s = np.maximum(old, np.abs(x).max((1, 2)).astype(F) / F(127))
                for h in range(self.h):
                    if held and s[h] > old[h]:
                        c = self.codes[n][at, h, :held].astype(F) * F(old[h] / s[h])
                        self.codes[n][at, h, :held] = np.rint(c).astype(np.int8)
                    new = np.rint(x[h] / s[h]) if s[h] > 0 else np.zeros_like(x[h])
                    self.codes[n][at, h, held:held + hi - lo] = np.clip(new, -127, 127).astype(np.int8)
                self.scale[n][at] = s

    def tokens(self, n, kv_len, table):
        """(values [kv_len][h][d] fp32, which of them the cache has)."""
        out, has = np.zeros((kv_len, self.h, self.d), F), np.zeros(kv_len, bool)
        for p in range(-(-kv_len // self.page)):
            at = self.place(table, p)
            if at is None:
                continue
            m = min(self.page, kv_len - p * self.page)
            s = slice(p * self.page, p * self.page + m)
            out[s] = (self.codes[n][at, :, :m].astype(F) * self.scale[n][at][:, None, None]).transpose(1, 0, 2)
            has[s] = True
        return out, has


def seen_by(n, kv_len, has, window, sinks):
    """[n][kv_len]: which tokens each of a sequence's n queries sees."""
    pos = kv_len - n + np.arange(n)[:, None]
    j = np.arange(kv_len)[None, :]
    seen = (j <= pos) & has[None, :]
    if window > 0:
        seen &= (pos - j < window) | (j < sinks)
    return seen


def attend(q, kv_len, k, v, seen, scale, gate=None):
    """o [q][h_q][d] in 64 bits for one sequence: q rows fp32, k and v [kv_len][h_kv][d], 0 where no query sees them."""
    n, h_q, d = q.shape
    G = h_q // k.shape[1]
    o = np.zeros((n, h_q, d))
    k, v = k.astype(np.float64), v.astype(np.float64)
    for h in range(h_q):
        with np.errstate(all="ignore"):
            a = np.where(seen, q[:, h].astype(np.float64) @ k[:, h // G].T * scale, -np.inf)
            top = a.max(1, keepdims=True, initial=-np.inf)
            p = np.exp(a - np.where(np.isneginf(top), 0, top))
            p[~seen] = 0
            total = p.sum(1, keepdims=True)
            o[:, h] = p @ v[:, h // G] / np.where(total == 0, 1, total)
    if gate is not None:
        o = o / (1 + np.exp(-gate.astype(np.float64)))
    return o


def normal_bf16(g, *shape, std=1.0):
    """(bf16 bits, their values in fp32)"""
    b = bf16.from_f32((g.standard_normal(shape) * std).astype(F))
    return b, bf16.to_f32(b)
