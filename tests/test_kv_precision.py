"""How far the two e4m3 terms of a bf16 query element, and of a weight, are off: the bounds that include/sixi_kv.h states,
on a restatement of the two splits (kv_reference.round_e4m3)."""

from __future__ import annotations

import numpy as np

import kv_reference as R

LO_QUERY, LO_WEIGHT = 16.0, 32.0  # how much finer the second term's unit is


def e4m3(x):
    return R.E4M3[R.round_e4m3(x)]


def split_query(x):
    """x in (-448, 448], the row's largest beyond 224."""
    hi = e4m3(x)
    return hi + e4m3((x - hi) * LO_QUERY) / LO_QUERY


def split_weight(w):
    """w in [0, 1], the tile's largest beyond 1/2: fp16, then its code rounded at bit 7, then the rest."""
    h = w.astype(np.float16)
    top = ((h.view(np.uint16).astype(np.uint32) + 0x40) & 0xFF80).astype(np.uint16).view(np.float16)
    rest = (h.astype(np.float64) - top.astype(np.float64)) * (256 * LO_WEIGHT)
    assert np.abs(rest).max() <= 448 and np.array_equal(e4m3(top.astype(np.float64) * 256), top.astype(np.float64) * 256)
    return top.astype(np.float64) + e4m3(rest) / (256 * LO_WEIGHT)


def test_query_elements():
    bits = np.arange(0x3000, 0x43E0, dtype=np.uint32) << 16  # bf16 values up to 448
    x = bits.view(np.float32).astype(np.float64)
    err = np.abs(split_query(x) - x)
    assert np.all(err[x >= 2.0 ** -6] == 0)  # exact above 1/14,336 of a largest element of 224
    assert err.max() <= 2.0 ** -14 and 2.0 ** -14 / 224 < 2.0 ** -21.8
    assert np.abs(split_query(-x) + x).max() == err.max()


def test_weights():
    w = np.concatenate([2.0 ** np.random.default_rng(1).uniform(-26, 0, 400_000), [1.0, 0.5, 2.0 ** -14, 0.0]])
    err = np.abs(split_weight(w) - w)
    big = w >= 2.0 ** -14
    assert np.all(err[big] <= w[big] * (2.0 ** -9 + 2.0 ** -11))  # within half a last place of 8 bits, 2^-8
    assert np.all(err[~big] <= 2.0 ** -23 + 2.0 ** -25)
    assert (2.0 ** -23 + 2.0 ** -25) / 0.5 < 2.0 ** -21.6  # of the largest, which is 1/2 at least
    assert split_weight(np.array([2.0 ** -22]))[0] > 0
