"""Drafted tokens written, rejected and written over: the cache's bytes and scales, and the attention over them, are those of
the definition (kv_reference.py). A rejected token leaves its mark where it raised its page's scale: the older tokens of
the page have been rounded at it, and it does not come down."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

import torch  # noqa: E402

import kv_reference as R  # noqa: E402
from test_gpu_kv import BF, F32, World, check_attend, host  # noqa: E402


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("page,heads,dim,start,drafts", [
    (16, 2, 64, [3, 12, 15, 16, 0], 4),     # within a page, up to its end, across it, at its beginning
    (32, 5, 96, [30, 31, 32, 33, 1], 8),
    (64, 1, 128, [40, 63, 64, 130, 5], 40),  # more rows a page than a warp takes
])
def test_rejected_drafts_are_written_over(dt, page, heads, dim, start, drafts):
    n, steps = 1 + drafts, 6
    w = World(51, [s + steps * n for s in start], page, heads, dim).fill(start)
    lens, raised = list(start), 0
    for _ in range(steps):
        x = w.rng.normal(size=(len(lens), n, heads, dim))
        wild = w.rng.random(len(lens)) < 0.5
        x[wild, -1] *= 2.0 ** w.rng.integers(6, 14)  # the last draft is far out
        k = torch.from_numpy(x).to(dt)
        v = torch.from_numpy(x[:, ::-1].copy() * 0.5).to(dt)
        at = [s + n for s in lens]
        before = w.rk.scale.copy()
        st = w.kv.append(k.view(-1, heads, dim).to("cuda:0"), v.view(-1, heads, dim).to("cuda:0"), w.batch([n] * len(lens), at))
        assert st.tolist() == [0] * len(lens)
        for s in range(len(lens)):
            w.rk.write(w.table[s], lens[s], host(k[s]))
            w.rv.write(w.table[s], lens[s], host(v[s]))
        raised += int((w.rk.scale > before * 32).sum())
        w.same_bytes()
        kept = w.rng.integers(0, n, len(lens))  # at least the first token, and never the last draft
        lens = [s + max(1, int(a)) for s, a in zip(lens, kept)]
    assert raised > 0
    check_attend(w, [1] * len(lens), heads * 2, dt, lens=lens)


def test_a_rejected_draft_leaves_the_scale_of_its_page():
    w = World(52, [16], 16, 1, 16)
    w.rk.scale[:], w.rv.scale[:] = 1.0, 1.0
    w.push()
    rows = np.ones((3, 1, 16))
    rows[1] = 2.0 ** -9
    rows[2] = 2.0 ** 12

    def append(x, length):
        t = torch.from_numpy(x).to(F32).to("cuda:0")
        assert w.kv.append(t, t, w.batch([len(x)], [length])).tolist() == [0]

    append(rows[:2], 2)
    page = w.table[0, 0]
    kept = R.E4M3[w.kv.k_pages[page, 0, :2].cpu().numpy()] * float(w.kv.k_scales[page, 0])
    assert np.array_equal(kept, rows[:2, 0])
    append(rows[2:], 3)  # a draft, rejected:
    append(rows[:1], 3)
    scale = float(w.kv.k_scales[page, 0])
    assert scale == 2.0 ** R.scale_exp(2.0 ** 12)  # still the draft's
    kept = R.E4M3[w.kv.k_pages[page, 0, :3].cpu().numpy()] * scale
    assert np.array_equal(kept, np.concatenate([rows[:1, 0], R.E4M3[R.round_e4m3(rows[1, 0] / scale)][None] * scale, rows[:1, 0]]))
    assert not np.array_equal(kept[1], rows[1, 0])
