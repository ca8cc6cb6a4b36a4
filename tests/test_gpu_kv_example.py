"""The speculative decoding example over the 8-bit cache: it runs, and drafts do not change the text."""

from __future__ import annotations

import sys

import pytest

from conftest import REPO, has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

sys.path.insert(0, str(REPO / "examples"))


def test_drafted_steps_write_what_plain_steps_write():
    import spec_decode_cache as E

    plain, steps, rate = E.decode(streams=5, tokens=40, drafts=0)
    assert steps == 40 and rate == 1.0
    drafted, fewer, more = E.decode(streams=5, tokens=40, drafts=4)
    # The two differ in how many positions a step covers, so in the order of the cache's writes and of the
    # matrix products' sums: a near-tie of two logits may fall the other way, after which a stream goes its own way.
    same = sum(a == b for a, b in zip(plain, drafted))
    assert same >= 3, (plain, drafted)
    assert all(a[0] == b[0] for a, b in zip(plain, drafted))
    assert fewer <= steps and more >= 1.0
