"""The cache's calls on thousands of sequences."""

from __future__ import annotations

import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

import torch  # noqa: E402

from sixi_smp.kv_cache import KvBatch, KvCache  # noqa: E402

DEV = torch.device("cuda:0")
TYPES = [torch.bfloat16, torch.float32]


def streams(n, dt):
    """n sequences of 9 tokens (zeros), a page each; the last token's queries."""
    kv = KvCache(n, 16, 1, 16, max_seqs=n, device=0)
    for t in (kv.k_pages, kv.v_pages):
        t.zero_()
    for t in (kv.k_scales, kv.v_scales):
        t.fill_(1.0)
    batch = KvBatch(torch.arange(n, dtype=torch.int32, device=DEV).view(n, 1), torch.arange(n + 1, device=DEV),
                    torch.full((n,), 9, dtype=torch.int32, device=DEV), n, 1)
    return kv, batch, torch.ones((n, 2, 16), dtype=dt, device=DEV)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [200, 700, 3000])
@pytest.mark.parametrize("where", [0, 0.5, 1])
def test_an_offset_out_of_order_is_reported_by_every_sequence(dt, n, where):
    kv, batch, q = streams(n, dt)
    assert kv.attend(q, batch)[2].eq(0).all()
    s = int(where * (n - 2)) + 1
    batch.offsets[s] += 5  # (the sequence before is longer then, and this one's end lies before its beginning)
    assert kv.attend(q, batch)[2].eq(2).all()
    batch.offsets[s] -= 5
    out, _, st = kv.attend(q, batch)
    assert st.eq(0).all() and out.eq(0).all()


def least_time(call, runs=5):
    times = []
    for _ in range(runs + 1):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times[1:])


@pytest.mark.parametrize("dt", TYPES)
def test_time_grows_with_the_sequences_not_with_their_square(dt):
    """Eight times the sequences: eight times the time at most, and as much again for what a time may be off."""
    t = []
    for n in (8_191, 65_528):
        kv, batch, q = streams(n, dt)
        out, lse, st = kv.attend(q, batch)
        t.append(least_time(lambda: kv.attend(q, batch, out=out, lse=lse, status=st)))
    assert t[1] <= 16 * t[0], t


@pytest.mark.parametrize("dt", TYPES)
def test_a_shorter_sequence_does_not_take_longer(dt):
    """Where units begin to be cut, time may not fall: half the tokens take no more than the whole, but for a fifth."""
    t = {}
    for n in (128, 256, 512, 1024):
        kv = KvCache(n // 16, 16, 3, 80, device=0)
        for p in (kv.k_pages, kv.v_pages):
            p.zero_()
        for p in (kv.k_scales, kv.v_scales):
            p.fill_(1.0)
        batch = KvBatch(torch.arange(n // 16, dtype=torch.int32, device=DEV).view(1, -1), torch.tensor([0, 2], device=DEV),
                        torch.tensor([n], dtype=torch.int32, device=DEV), 2, 2)
        q = torch.ones((2, 21, 80), dtype=dt, device=DEV)
        out, lse, st = kv.attend(q, batch)
        call = torch.cuda.CUDAGraph()
        with torch.cuda.graph(call):
            for _ in range(20):
                kv.attend(q, batch, out=out, lse=lse, status=st)
        t[n] = least_time(call.replay)
    assert all(t[n] <= 1.2 * t[2 * n] for n in (128, 256, 512)), t
