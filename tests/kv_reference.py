"""The 8-bit paged key/value cache in 64 bits (numpy), from its definition: the tests' reference."""

from __future__ import annotations

import math

import numpy as np

# the 256 e4m3 values by their bits: sign, 4 exponent bits (bias 7), 3 mantissa bits, 0x7F and 0xFF NaN
E4M3 = np.array([(-1.0) ** (b >> 7) * (((b & 7) / 8) * 2.0 ** -6 if (b >> 3) & 15 == 0
                                       else (1 + (b & 7) / 8) * 2.0 ** (((b >> 3) & 15) - 7)) for b in range(256)])
E4M3[0x7F] = E4M3[0xFF] = np.nan


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """Bits of the nearest e4m3 value, ties to the even mantissa, beyond 448 to 448."""
    mags = E4M3[:0x7F]
    a = np.minimum(np.abs(x), 448.0)
    hi = np.clip(np.searchsorted(mags, a), 0, 0x7E)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - mags[lo], mags[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return (pick | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def scale_exp(amax: float) -> int:
    e = -126
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def inv_freq(rot, base=10000.0, scaling="none", factor=1.0, original_max_position=0, beta_fast=32.0, beta_slow=1.0):
    i = np.arange(rot // 2)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        at = lambda t: rot * math.log(original_max_position / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(at(beta_fast))), min(rot - 1, math.ceil(at(beta_slow)))
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return f / factor * r + f * (1 - r), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def rotate(x, pos, freq, amp, layout="half", inverse=False):
    """x [tokens, heads, dim] (64 bits) turned by pos [tokens]."""
    rot = 2 * len(freq)
    ang = np.asarray(pos, np.float64)[:, None] * freq[None, :]
    c, s = amp * np.cos(ang)[:, None, :], (-amp if inverse else amp) * np.sin(ang)[:, None, :]
    y = np.array(x, np.float64)
    sel = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = x[..., sel[0]], x[..., sel[1]]
    y[..., sel[0]], y[..., sel[1]] = a * c - b * s, b * c + a * s
    return y


class Cache:
    """Pages of bytes and scale exponents, written token range by token range."""

    def __init__(self, n_pages, heads, page, dim, rng=None):
        self.page = page
        # what unwritten memory holds is anything, NaN bytes and huge scales included
        self.bytes = np.full((n_pages, heads, page, dim), 0x7F, np.uint8)
        self.scale = np.full((n_pages, heads), 1e30, np.float32)
        if rng is not None:
            self.bytes[:] = rng.integers(0, 256, self.bytes.shape)

    def write(self, table, start, x):
        """x [n, heads, dim] at positions start..; returns whether something was not finite."""
        n, heads, _ = x.shape
        bad = False
        for first in range(start // self.page * self.page, start + n, self.page):
            p = int(table[first // self.page])
            lo, hi = max(first, start), min(first + self.page, start + n)
            for h in range(heads):
                rows = x[lo - start:hi - start, h].astype(np.float64)
                bad |= not np.isfinite(rows).all()
                rows = np.where(np.isnan(rows), 0.0, rows)
                fin = np.abs(rows[np.isfinite(rows)])
                s = 2.0 ** scale_exp(fin.max() if fin.size else 0.0)
                if lo > first:
                    old = float(self.scale[p, h])
                    if s > old:
                        held = E4M3[self.bytes[p, h, :lo - first]] * old
                        self.bytes[p, h, :lo - first] = round_e4m3(held / s)
                    s = max(s, old)
                self.scale[p, h] = s
                self.bytes[p, h, lo - first:hi - first] = round_e4m3(np.clip(rows / s, -448, 448))
        return bad

    def values(self, table, h, length):
        ids = np.asarray(table[: -(-length // self.page)], np.int64)
        v = E4M3[self.bytes[ids, h]] * self.scale[ids, h].astype(np.float64)[:, None, None]
        return v.reshape(-1, v.shape[-1])[:length]


def attend(cache_k: Cache, cache_v: Cache, table, length, q, scale, window=0, causal=True):
    """q [n, heads_q, dim] (64 bits) at the last n positions: (out, lse, sum of p|v|, and the largest
    sum of |q||k| of a score, times scale)."""
    n, hq, dim = q.shape
    hk = cache_k.bytes.shape[1]
    out, lse, mag = np.zeros((n, hq, dim)), np.full((n, hq), -np.inf), np.zeros((n, hq, dim))
    reach = 0.0
    t = np.arange(length)
    for h in range(hk):
        k, v = cache_k.values(table, h, length), cache_v.values(table, h, length)
        for i in range(n):
            p = length - n + i
            ok = np.ones(length, bool) if not causal else t <= p
            if window:
                ok &= t > p - window
            if not ok.any():
                continue
            for j in range(h * (hq // hk), (h + 1) * (hq // hk)):
                s = (k[ok] @ q[i, j]) * scale
                reach = max(reach, float((np.abs(k[ok]) @ np.abs(q[i, j])).max() * abs(scale)))
                m = s.max()
                w = np.exp(s - m)
                lse[i, j] = m + math.log(w.sum())
                w /= w.sum()
                out[i, j] = w @ v[ok]
                mag[i, j] = w @ np.abs(v[ok])
    return out, lse, mag, reach
