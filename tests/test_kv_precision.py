"""How far the two e4m3 terms of a bf16 query element are off: the bound that the kernel's comment states, on a restatement
of the split (kv_reference.round_e4m3)."""

from __future__ import annotations

import numpy as np

import kv_reference as R

LO_QUERY = 16.0  # how much finer the second term's unit is


def e4m3(x):
    return R.E4M3[R.round_e4m3(x)]


def split_query(x):
    """x in (-448, 448], the row's largest beyond 224."""
    hi = e4m3(x)
    return hi + e4m3((x - hi) * LO_QUERY) / LO_QUERY


def test_query_elements():
    bits = np.arange(0x3000, 0x43E0, dtype=np.uint32) << 16  # bf16 values up to 448
    x = bits.view(np.float32).astype(np.float64)
    err = np.abs(split_query(x) - x)
    assert np.all(err[x >= 2.0 ** -6] == 0)  # exact above 1/14,336 of a largest element of 224
    assert err.max() <= 2.0 ** -14 and 2.0 ** -14 / 224 < 2.0 ** -21.8
    assert np.abs(split_query(-x) + x).max() == err.max()
