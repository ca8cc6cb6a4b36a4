"""Attention over the 8-bit cache at the ends of its range, against the definition in 64 bits (kv_reference.py).

Tolerances as in test_gpu_kv.py: a score errs by (dim + 8) u R at most, R the row's largest sum of scale |q| |k|; a
weight by a factor e^(2 err) and, with bf16 queries, by 2^-9 (its two terms) + 2^-11 (its fp16 form on the way); the output
by its type (u = 2^-24, b = 2^-8)."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

import torch  # noqa: E402

import kv_reference as R  # noqa: E402
from test_gpu_kv import B, BF, DEV, F32, U, World, host  # noqa: E402


def contents(w, k, v):
    """The cache's contents: k, v [tokens, heads, dim] of its one sequence, on both sides."""
    w.rk.write(w.table[0], 0, k)
    w.rv.write(w.table[0], 0, v)
    w.push()
    return w


def check(w, q, scale=None, window=0):
    """q [new, query heads, dim] (host, of its type) over the cache's one sequence."""
    n, length = q.shape[0], w.lens[0]
    sc = w.dim ** -0.5 if scale is None else scale
    out, lse, st = w.kv.attend(q.to(DEV), w.batch([n]), scale=scale, window=window)
    assert st.tolist() == [0]
    ro, rl, mag, reach = R.attend(w.rk, w.rv, w.table[0], length, host(q), sc, window)
    bf = q.dtype == BF
    err = (w.dim + 8) * U * reach
    weights = 2 * err + (length / 16 + 64) * U + (2.0 ** -9 + 2.0 ** -11 if bf else 0)
    tol = weights * mag * math.e + (B if bf else 2 * U) * np.abs(ro) + 1e-30
    got, gl = host(out), host(lse)
    assert np.all(np.abs(got - ro) <= tol), float((np.abs(got - ro) / tol).max())
    assert np.all(np.abs(gl - rl) <= err + (length / 16 + 64) * U + 4 * U * np.abs(rl))


# ---------------------------------------------------------------------------------------------
# scores: queries and keys whose magnitudes cancel


@pytest.mark.parametrize("heads,group,dim,page", [(1, 4, 128, 64), (2, 8, 64, 16), (1, 20, 256, 32), (1, 64, 80, 128)])
@pytest.mark.parametrize("mag", [1e-28, 1e-32, 1e-36, 1e-20, 1e20, 1e30, 1e33])
def test_small_queries_on_large_keys_and_the_other_way_round(mag, heads, group, dim, page):
    w = World(41, [400], page, heads, dim)
    k = w.rng.normal(size=(400, heads, dim)) / mag
    contents(w, np.clip(k, -3e38, 3e38), w.rng.normal(size=(400, heads, dim)))
    for n in (1, 3):
        check(w, torch.from_numpy(w.rng.normal(size=(n, heads * group, dim)) * mag).to(BF))


@pytest.mark.parametrize("mag", [1e-32, 1e-28, 1e-20, 1e20, 1e28])
def test_small_queries_on_large_keys_in_fp32(mag):
    w = World(42, [400], 64, 2, 64)
    contents(w, w.rng.normal(size=(400, 2, 64)) / mag, w.rng.normal(size=(400, 2, 64)))
    check(w, torch.from_numpy(w.rng.normal(size=(3, 8, 64)) * mag).to(F32))


def test_small_queries_over_pages_of_very_different_scales():
    """Keys of some pages 2^90 times others', values too: the maxima of weight times value scale come from other tokens."""
    w = World(43, [96], 16, 1, 64)
    mag = np.repeat(2.0 ** np.array([90, 0, 85, 20, 89, -10]), 16)[:, None, None]
    contents(w, w.rng.normal(size=(96, 1, 64)) * mag,
             w.rng.normal(size=(96, 1, 64)) * np.repeat(2.0 ** np.array([0, -12, 9, -30, 3, 20]), 16)[:, None, None])
    check(w, torch.from_numpy(w.rng.normal(size=(4, 2, 64)) * 2.0 ** -90).to(BF))


@pytest.mark.parametrize("scale,mag", [(1e-30, 1e30), (1e-38, 1e36), (1e30, 1e-30), (3e38, 1e-38)])
def test_scales_that_cancel_the_queries(scale, mag):
    w = World(44, [300], 32, 1, 128)
    contents(w, w.rng.normal(size=(300, 1, 128)) * 0.1, w.rng.normal(size=(300, 1, 128)))
    check(w, torch.from_numpy(w.rng.normal(size=(2, 8, 128)) * mag).to(BF), scale=scale)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("heads,group,dim,page", [(1, 16, 64, 64), (2, 4, 128, 16), (1, 40, 128, 32), (1, 32, 256, 128)])
def test_scores_beyond_24_bits(dt, heads, group, dim, page):
    """One token far above the others, by scores from 20 to 10^29 whose roundings are whole numbers or more: its weight is
    1 and theirs 0 all the same. A score here is one product, so lse is off by the roundings of its factors only."""
    n, at = 300, 137
    w = World(45, [n], page, heads, dim)
    k = np.zeros((n, heads, dim))
    k[:, :, 0] = -1.0
    k[at, :, 0] = 1.0
    contents(w, k, w.rng.normal(size=(n, heads, dim)))
    q = torch.zeros((5, heads * group, dim))
    q[:, :, 0] = torch.from_numpy(10.0 ** w.rng.uniform(2.5, 30, size=(5, heads * group)))
    q = q.to(dt)
    out, lse, _ = w.kv.attend(q.to(DEV), w.batch([5]))
    want = np.repeat(np.stack([w.rv.values(w.table[0], h, n)[at] for h in range(heads)]), group, 0)[None]
    b = B if dt == BF else 4 * U
    assert np.all(np.abs(host(out) - want) <= b * np.abs(want) + 1e-9)
    score = host(q)[:, :, 0] * dim ** -0.5
    assert np.all(np.abs(host(lse) - score) <= 6 * U * score)


@pytest.mark.parametrize("mag", [1e-36, 1e-33, 1e33, 1e36, 1e37])
def test_queries_near_the_ends_of_fp32(mag):
    """A product of a query element and a cached byte may pass fp32's range although the score does not."""
    w = World(46, [400], 64, 2, 128)
    k = w.rng.normal(size=(400, 2, 128)) / mag
    contents(w, np.clip(k, -3e38, 3e38), w.rng.normal(size=(400, 2, 128)))
    check(w, torch.from_numpy(w.rng.normal(size=(3, 8, 128)) * mag).to(F32))


# ---------------------------------------------------------------------------------------------
# bits: bf16 queries and weights are split into two e4m3 terms


@pytest.mark.parametrize("dim,group", [(64, 8), (128, 40), (256, 32)])
def test_small_elements_of_a_query_keep_their_bits(dim, group):
    """A query whose largest element, 900 to 14,000 times the others, meets keys that are zero there: the scores come from
    the others alone, exactly."""
    w = World(47, [200], 32, 1, dim)
    k = w.rng.normal(size=(200, 1, dim)) * 20
    k[:, :, 0] = 0.0
    contents(w, k, w.rng.normal(size=(200, 1, dim)))
    q = w.rng.normal(size=(3, group, dim)) * 0.5
    q[:, :, 0] = 500.0 * 2.0 ** w.rng.uniform(0, 4, size=(3, group))
    q[:, :, 1:] *= (np.abs(q[:, :, 1:]) > q[:, :, :1] / 13_000)
    check(w, torch.from_numpy(q).to(BF), scale=1.0 / (20 * dim ** 0.5))


@pytest.mark.parametrize("group", [8, 16, 32, 40, 64])
def test_weights_above_2_13_of_the_largest_keep_8_bits(group):
    """Two tokens, the heavier one's value zero: the output is the lighter one's weight, here 2^-13 to 2^-14 of the largest,
    times its values. Eight significands of those tell within which bounds the weight is, whatever the output's type rounds
    away. It may be off by 2^-9 (its two terms) + 2^-11 (its fp16 form on the way), and its exponent by the roundings of
    two scores below 32 and of the exponential."""
    w = World(48, [2], 16, 1, 64)
    k = np.zeros((2, 1, 64))
    k[0, 0, 0] = k[1, 0, 1] = 1.0
    k[1, 0, 2] = 2.0 ** -4
    v = np.zeros((2, 1, 64))
    v[1, 0] = 1.0 + np.arange(64) % 8 / 8
    contents(w, k, v)
    q = np.zeros((64, group, 64))
    q[:, :, 0] = 16.0
    q[:, :, 1] = 16.0 - w.rng.uniform(9.1, 9.6, size=(64, group))
    q[:, :, 2] = w.rng.uniform(0, 0.5, size=(64, group))
    q = torch.from_numpy(q).to(BF)
    gap = host(q)[:, :, 0] - host(q)[:, :, 1] - host(q)[:, :, 2] / 16
    out = np.concatenate([host(w.kv.attend(q[i:i + 1].to(DEV), w.batch([1]), scale=1.0)[0]) for i in range(64)])
    half = 2.0 ** (np.floor(np.log2(out)) - 8)  # half a last place
    at_least, at_most = ((out - half) / v[1, 0]).max(-1), ((out + half) / v[1, 0]).min(-1)
    want, off = 1.0 / (1.0 + np.exp(gap)), 2.0 ** -9 + 2.0 ** -11 + 100 * U
    assert np.all(want >= at_least / (1 + off)) and np.all(want <= at_most / (1 - off))
