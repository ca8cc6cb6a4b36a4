"""Attention over the 8-bit cache at the ends of its range."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

import torch  # noqa: E402

from test_gpu_kv import B, BF, DEV, F32, U, World, host  # noqa: E402


def contents(w, k, v):
    """The cache's contents: k, v [tokens, heads, dim] of its one sequence, on both sides."""
    w.rk.write(w.table[0], 0, k)
    w.rv.write(w.table[0], 0, v)
    w.push()
    return w


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("heads,group,dim,page", [(1, 16, 64, 64), (2, 4, 128, 16), (1, 40, 128, 32), (1, 32, 256, 128)])
def test_scores_beyond_24_bits(dt, heads, group, dim, page):
    """One token far above the others, by scores from 12 to 10^29 whose roundings are whole numbers or more: its weight is
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
