"""Calls on a named stream that is not the current one: their results do not land in memory that the current stream still
uses, and what they were given is not handed out again before they have read it."""

from __future__ import annotations

import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

import numpy as np  # noqa: E402
import torch  # noqa: E402

import sixi_smp as S  # noqa: E402
from sixi_smp.kv_cache import KvBatch, KvCache, Rope  # noqa: E402

DEV = torch.device("cuda:0")
DELAY = 200_000_000  # cycles: a tenth of a second


def cache_calls():
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    n, heads, dim = 512, 4, 64
    q = torch.randn((n, heads, dim), device=DEV, generator=g).to(torch.bfloat16)
    kv = KvCache(40, 16, heads, dim, device=0, max_seqs=4)
    batch = KvBatch(torch.arange(32, dtype=torch.int32, device=DEV).view(1, 32), torch.tensor([0, n], device=DEV),
                    torch.tensor([n], dtype=torch.int32, device=DEV), n, n)
    rope, pos = Rope(dim, device=0), torch.arange(n, dtype=torch.int32, device=DEV)
    kv.append(q, q, batch)
    return {"attend": (q, lambda x, s: kv.attend(x, batch, stream=s)[0]),
            "apply": (q, lambda x, s: rope.apply(x, pos, stream=s)),
            "read": (q, lambda x, s: kv.read(batch, stream=s)[0])}


@pytest.mark.parametrize("name", ["attend", "apply", "read"])
def test_results_do_not_land_in_the_current_streams_memory(name):
    x, call = cache_calls()[name]
    want = call(x, None).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(DELAY)
    held = [torch.empty_like(want).fill_(7.0) for _ in range(4)]  # still to be written when their memory is given back
    del held
    got = call(x, side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["attend", "apply"])
def test_what_a_call_was_given_is_not_handed_out_again(name):
    x, call = cache_calls()[name]
    want = call(x, None).clone()
    side = torch.cuda.Stream()
    mine = x.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(DELAY)
    got = call(mine, side)
    del mine
    again = [torch.empty_like(x).fill_(7.0) for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(again) == 4


@pytest.mark.parametrize("delayed", ["current", "named"])
def test_sampler_candidates_on_a_named_stream(delayed):
    """Its outputs are filled before the call: on the stream that the call runs on."""
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    logits = torch.randn((32, 4096), device=DEV, generator=g)
    smp = S.Sampler(0, 32, 4096)
    params = torch.from_numpy(S.make_params(32, temperature=0.7, top_k=20).view(np.uint8)).to(DEV)
    want = [t.clone() for t in smp.candidates(logits, params, max_out=32)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.current_stream() if delayed == "current" else side):
        torch.cuda._sleep(DELAY)
    mine = logits.clone() if delayed == "named" else logits
    torch.cuda.current_stream().synchronize() if delayed == "named" else None
    got = smp.candidates(mine, params, max_out=32, stream=side)
    del mine
    again = torch.empty_like(logits).fill_(7.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and again is not None
    smp.close()
