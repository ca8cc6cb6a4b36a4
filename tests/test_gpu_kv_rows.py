"""Attention with bf16 queries at every number of rows that a row tile may have: the new tokens of a sequence times the
query heads of a key head, in blocks of 8 up to 64 (32 for heads beyond 128 elements), one row short of them and one more."""

from __future__ import annotations

import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

from test_gpu_kv import BF, World, check_attend  # noqa: E402


@pytest.mark.parametrize("dim", [128, 80, 192])
@pytest.mark.parametrize("rows", [7, 9, 16, 17, 23, 24, 25, 33, 40, 41, 47, 48, 49, 55, 56, 57, 63, 64, 65, 72, 96, 112])
def test_rows_of_a_tile(rows, dim):
    w = World(61, [300, 130, 64], 32, 2, dim).fill()
    check_attend(w, [rows, 1, 2], 2, BF)


@pytest.mark.parametrize("group", [3, 6, 7, 12, 14, 24, 28])
@pytest.mark.parametrize("dim,window", [(64, 0), (128, 50), (256, 0)])
def test_rows_of_a_tile_with_several_heads(group, dim, window):
    w = World(62, [200, 400], 16, 1, dim).fill()
    check_attend(w, [8, 3], group, BF, window=window)
