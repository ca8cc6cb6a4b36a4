"""The speculative decoding example where drafts are accepted: a small vocabulary, whose text repeats itself."""

from __future__ import annotations

import sys

import pytest

from conftest import REPO, has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

sys.path.insert(0, str(REPO / "examples"))


@pytest.mark.parametrize("vocab,seed", [(16, 0), (32, 1), (64, 0)])
def test_accepted_drafts_save_steps(vocab, seed):
    import spec_decode_cache as E

    plain, steps, rate = E.decode(streams=5, tokens=64, drafts=0, vocab=vocab, seed=seed)
    assert steps == 64 and rate == 1.0 and all(len(t) == 64 for t in plain)
    drafted, fewer, more = E.decode(streams=5, tokens=64, drafts=4, vocab=vocab, seed=seed)
    assert fewer < 0.9 * steps and more > 1.2
    assert all(len(t) == 64 for t in drafted)
    assert sum(a == b for a, b in zip(plain, drafted)) >= 4  # (a near-tie of two logits may fall the other way)
