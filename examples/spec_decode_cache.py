"""Speculative decoding over the 8-bit paged cache: a small random transformer, the suffix drafter and the verifier.

Every step runs, for all streams at once, what a serving loop runs per layer and then per step:

    cache.append     the step's keys (turned by their positions) and values, 1 + k tokens a stream
    cache.attend     their queries over everything cached
    ... residual, next layer; logits of every position ...
    suffix_draft     k tokens that continue the stream the way its own history once went on
    verify           greedy match of the drafts against the logits, and the token after the last match

and then moves each stream's length on by what was accepted: rejected drafts stay behind the length and
are written over. The cache is paged; pages are dealt to streams as they grow, out of one pool.

    python examples/spec_decode_cache.py [--streams 8] [--tokens 48] [--drafts 4] [--vocab 4096] [--plain]

--plain drafts nothing and verifies one token a step. Both choose the same tokens but for near-ties of two
logits: a draft changes how many positions a step covers, so the order in which products are summed, and
a rejected draft that was the largest of its page leaves the page's scale raised, and the page's older
tokens rounded at that.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "sixi-asi_b200"))

import sixi_smp as S  # noqa: E402
from sixi_smp.kv_cache import KvBatch, KvCache, Rope  # noqa: E402


class Model:
    """Random weights, cached keys and values in 8 bits; logits of the batch's positions."""

    def __init__(self, vocab=4096, layers=2, q_heads=16, kv_heads=4, dim=64, page=32, pages=512, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        width = q_heads * dim

        def weight(*shape):
            return (torch.randn(shape, device="cuda", generator=g) / shape[0] ** 0.5).to(torch.bfloat16)

        self.vocab, self.q_heads, self.kv_heads, self.dim = vocab, q_heads, kv_heads, dim
        self.embed = weight(vocab, width) * vocab ** 0.5
        self.head = weight(width, vocab)
        self.q = [weight(width, q_heads * dim) for _ in range(layers)]
        self.kv = [weight(width, 2 * kv_heads * dim) for _ in range(layers)]
        self.out = [weight(q_heads * dim, width) for _ in range(layers)]
        self.rope = Rope(rot_dim=dim, base=10000.0)
        self.caches = [KvCache(pages, page, kv_heads, dim) for _ in range(layers)]

    def logits(self, tokens, batch: KvBatch):
        n = tokens.shape[0]
        x = self.embed[tokens.long()]
        statuses = []
        for q, kv, out, cache in zip(self.q, self.kv, self.out, self.caches):
            h = x / x.float().square().mean(-1, keepdim=True).add(1e-6).sqrt().to(x.dtype)
            kvs = (h @ kv).view(n, 2, self.kv_heads, self.dim)
            statuses.append(cache.append(kvs[:, 0], kvs[:, 1], batch, rope=self.rope))
            a, _, st = cache.attend((h @ q).view(n, self.q_heads, self.dim), batch, rope=self.rope)
            statuses.append(st)
            x = x + a.reshape(n, -1) @ out
        return (x @ self.head).float(), torch.stack(statuses).amax(0)


class Pages:
    """Pages of one pool dealt to streams as they grow."""

    def __init__(self, streams, pages, page, longest):
        self.free = list(range(pages))[::-1]
        self.page = page
        self.table = np.full((streams, -(-longest // page)), -1, np.int32)
        self.held = [0] * streams

    def reach(self, lens):
        for s, n in enumerate(lens):
            while self.held[s] * self.page < n:
                self.table[s, self.held[s]] = self.free.pop()
                self.held[s] += 1
        return torch.from_numpy(self.table).cuda()


def decode(streams=8, tokens=48, drafts=4, prompt=24, seed=0, vocab=4096):
    """(generated tokens per stream, steps, tokens per step of a stream that is not done). Greedy: drafts change the
    text by near-ties only."""
    model = Model(vocab=vocab, seed=seed)
    rng = np.random.default_rng(seed)
    hist = [list(rng.integers(0, model.vocab, prompt // 2)) * 2 for _ in range(streams)]
    start = len(hist[0])
    stop = start + tokens
    pages = Pages(streams, 512, 32, stop + drafts)
    smp = S.Sampler(0, streams * (drafts + 1), model.vocab)
    params = torch.from_numpy(S.make_params(streams, temperature=0.0).view(np.uint8)).cuda()

    # the prompts but for their last token, in one call
    n = start - 1
    off = torch.arange(streams + 1, dtype=torch.int64).cuda() * n
    lens = torch.full((streams,), n, dtype=torch.int32).cuda()
    flat = torch.tensor([t for h in hist for t in h[:-1]], dtype=torch.int32).cuda()
    _, st = model.logits(flat, KvBatch(pages.reach([n] * streams), off, lens, streams * n, n))
    assert (st == 0).all()

    steps = written = worked = 0
    while min(len(h) for h in hist) < stop:
        k = drafts
        if k:
            offs = np.concatenate([[0], np.cumsum([len(h) for h in hist])]).astype(np.int64)
            d, _ = smp.suffix_draft(torch.tensor([t for h in hist for t in h], dtype=torch.int32).cuda(),
                                    torch.from_numpy(offs).cuda(), k)
            guess = d.cpu().numpy()
            guess = np.where(guess < 0, 0, guess).astype(np.int32)  # streams without a proposal draft token 0
        else:
            guess = np.zeros((streams, 0), np.int32)
        # 1 + k tokens a stream: the last one that is certain, then the drafts
        feed = np.concatenate([np.array([[h[-1]] for h in hist], np.int32), guess], 1)
        cached = [len(h) + k for h in hist]
        off = torch.arange(streams + 1, dtype=torch.int64).cuda() * (1 + k)
        batch = KvBatch(pages.reach(cached), off, torch.tensor(cached, dtype=torch.int32).cuda(), streams * (1 + k), 1 + k)
        logits, st = model.logits(torch.from_numpy(feed.reshape(-1)).cuda(), batch)
        assert (st == 0).all()
        if k:
            v = smp.verify(logits, torch.from_numpy(guess).cuda(), params)
            out, count = v["tokens"].cpu().numpy(), v["n_tokens"].cpu().numpy()
        else:
            tok, _ = smp.greedy_argmax(logits)
            out, count = tok.cpu().numpy()[:, None], np.ones(streams, np.int64)
        for s in range(streams):  # a stream's length moves on by what was accepted, up to the end of its text
            if len(hist[s]) < stop:
                written, worked = written + int(count[s]), worked + 1
                hist[s] = (hist[s] + [int(t) for t in out[s, : count[s]]])[:stop]
        steps += 1
    text = [h[start:] for h in hist]
    smp.close()
    return text, steps, written / worked


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--streams", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=4096, help="a small one repeats itself, so that drafts are accepted")
    ap.add_argument("--plain", action="store_true")
    a = ap.parse_args()
    text, steps, rate = decode(a.streams, a.tokens, 0 if a.plain else a.drafts, vocab=a.vocab)
    print(f"{a.streams} streams x {a.tokens} tokens in {steps} steps, {rate:.2f} tokens a step")
    print("stream 0:", text[0])


if __name__ == "__main__":
    main()
