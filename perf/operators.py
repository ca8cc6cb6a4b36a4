"""Cases of the 8-bit paged key/value cache: rotary positions, writing and reading the cache, and
attention over it, as a serving loop around the sampler and the speculative verifier calls them.

`run` computes a case either with the plain form (elementary torch operations in 32 bits) or, where
`own` is set, with the library's entry points (sixi_smp.kv_cache).

The cache: pages of `page` tokens, [n_pages, kv_heads, page, head_dim] bytes in e4m3, with one
power-of-two fp32 scale per page and head: 2^e with the least e >= -126 such that the largest
magnitude that was written to the page is at most 448 * 2^e. A call that adds tokens to a page which
holds older ones keeps the larger of the old and the new scale; where it grows, the older values
are rounded again at the new one. Sequences own pages through a page table; a batch describes, for
each sequence, the last n_s of its lens_s positions: the tokens to write, to read, or whose queries
attend.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SZ = {"bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------
# cases


def _rope_case(tokens, heads, dim, rot, layout, dtype, scaling, factor, max_pos, inverse, **kw):
    return dict(op="rope", tokens=tokens, heads=heads, dim=dim, rot=rot, layout=layout, dtype=dtype,
                scaling=scaling, factor=factor, max_pos=max_pos, inverse=inverse, **kw)


def _append_case(seqs, new_min, new_max, ctx_max, kv_heads, dim, page, dtype, rot, **kw):
    return dict(op="append", seqs=seqs, new_min=new_min, new_max=new_max, ctx_max=ctx_max,
                kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, rot=rot, **kw)


def _attend_case(seqs, new_min, new_max, len_min, len_max, q_heads, kv_heads, dim, page, dtype, window, rot, **kw):
    return dict(op="attend", seqs=seqs, new_min=new_min, new_max=new_max, len_min=len_min, len_max=len_max,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, window=window, rot=rot, **kw)


def listed():
    return [
        # one decode step of a few streams: queries and keys of 5 tokens, interleaved pairs, fp32
        _rope_case(5, 12, 64, 64, "interleaved", "f32", "none", 1.0, 4096, False, name="rope_step"),
        # half of an odd-sized head turned back (the gradient, or keys moved to other positions)
        _rope_case(777, 17, 160, 80, "half", "bf16", "linear", 4.0, 32768, True, name="rope_partial_inverse"),
        # prompts of a batch at once, positions far past the trained length (yarn)
        _rope_case(16384, 40, 128, 128, "half", "bf16", "yarn", 8.0, 262144, False, name="rope_prompt"),
        # one token for each of 64 streams: what every decode step writes
        _append_case(64, 1, 1, 8192, 8, 128, 64, "bf16", 128, name="append_decode"),
        # drafted tokens of 37 streams, ragged, small pages, odd heads, fp32 keys without rotation
        _append_case(37, 1, 9, 700, 5, 96, 16, "f32", 0, name="append_drafts"),
        # prompts: 5 sequences of up to 8,000 tokens, fused with the rotation of their keys
        _append_case(5, 500, 8000, 300, 8, 128, 64, "bf16", 128, name="append_prompt"),
        # the smallest serving call: one stream, one token, a short context
        _attend_case(1, 1, 1, 700, 700, 32, 8, 128, 64, "bf16", 0, 0, name="attend_one"),
        # a decode step of 64 streams with ragged contexts, queries rotated on the way in
        _attend_case(64, 1, 1, 500, 16000, 32, 8, 128, 64, "bf16", 0, 128, name="attend_decode"),
        # verification of 8 drafts + 1 for 32 streams (the verifier's batch), small pages
        _attend_case(32, 9, 9, 300, 8000, 64, 8, 128, 16, "bf16", 0, 0, name="attend_verify"),
        # two very long contexts, one token each: few rows, a long axis
        _attend_case(2, 1, 1, 200001, 262144, 32, 4, 128, 128, "bf16", 0, 0, name="attend_long"),
        # chunks of prompts on top of cached prefixes, sliding window, wide heads
        _attend_case(3, 300, 2048, 2500, 9000, 16, 4, 256, 64, "bf16", 4096, 0, name="attend_chunk"),
        # fp32 queries, 7 query heads to a key head, a head size that is no power of two
        _attend_case(6, 1, 4, 33, 3000, 21, 3, 80, 32, "f32", 0, 0, name="attend_f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    most = [max(work(c)[key] for c in listed()) for key in ("bytes", "flops")]
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return c


def _draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "rope":
        dim = 16 * rng.randint(2, 16)
        rot = rng.choice([dim, 2 * rng.randint(4, dim // 2)])
        return _rope_case(_log_int(rng, 1, 12000), _log_int(rng, 1, 40), dim, rot,
                          rng.choice(["half", "interleaved"]), dtype, rng.choice(["none", "linear", "ntk", "yarn"]),
                          rng.choice([2.0, 4.0, 8.0]), _log_int(rng, 100, 500000), rng.random() < 0.3)
    page = rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    if op == "append":
        if rng.random() < 0.5:  # a step: few tokens for many streams
            a = rng.randint(1, 12)
            seqs, new = _log_int(rng, 1, 256), (rng.randint(1, a), a)
        else:  # prompts
            a = _log_int(rng, 64, 8000)
            seqs, new = rng.randint(1, 5), (max(1, a // rng.randint(1, 16)), a)
        return _append_case(seqs, new[0], new[1], _log_int(rng, 1, 4000), rng.randint(1, 8), dim, page, dtype,
                            rng.choice([0, dim, dim // 2]))
    kv = rng.randint(1, 8)
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16]) if kv <= 4 else rng.choice([1, 2, 4, 5, 7, 8])
    kind = rng.choice(["decode", "decode", "verify", "long", "chunk"])
    window = rng.choice([0, 0, 0, _log_int(rng, 100, 8000)])
    rot = rng.choice([0, 0, dim])
    if kind == "decode":
        hi = _log_int(rng, 20, 16000)
        seqs, new, lens = _log_int(rng, 1, 64), (1, 1), (max(1, hi // rng.randint(1, 30)), hi)
    elif kind == "verify":
        hi, a = _log_int(rng, 40, 8000), rng.randint(2, 16)
        seqs, new, lens = _log_int(rng, 1, 32), (rng.randint(1, a), a), (max(16, hi // rng.randint(1, 30)), hi)
    elif kind == "long":
        hi = _log_int(rng, 20000, 200000)
        seqs, new, lens = rng.randint(1, 2), (1, rng.choice([1, 1, 5])), (hi // 2, hi)
    else:
        hi = _log_int(rng, 300, 8000)
        a = _log_int(rng, 17, min(1500, hi))
        seqs, new, lens = rng.randint(1, 3), (max(1, a // 3), a), (max(a, hi // 2), hi)
        dtype = "bf16"
    if dtype == "f32":
        lens = (max(1, lens[0] // 8), max(16, lens[1] // 8))
    return _attend_case(seqs, new[0], new[1], lens[0], lens[1], kv * group, kv, dim, page, dtype, window, rot)


def _spread(lo, hi, n, phase):
    """n whole numbers over [lo, hi], spread over their logarithm, the last of them hi; the same for every seed."""
    out = []
    for i in range(n):
        u = (i * 0.6180339887498949 + phase) % 1.0
        out.append(min(hi, max(lo, int(round(math.exp(math.log(lo) + u * (math.log(hi + 1) - math.log(lo))))))))
    out[-1] = hi
    return out


def _lengths(c):
    """(new tokens, lengths with them) of each sequence of an append or attend case."""
    new = _spread(c["new_min"], c["new_max"], c["seqs"], 0.31)
    if c["op"] == "append":
        ctx = _spread(1, c["ctx_max"] + 1, c["seqs"], 0.77)
        return new, [a + b - 1 for a, b in zip(new, ctx)]
    lens = _spread(c["len_min"], c["len_max"], c["seqs"], 0.77)
    return [min(a, b) for a, b in zip(new, lens)], lens


def _pairs(c):
    """(row, token) pairs that attention computes, and the cached tokens that some row of each sequence reads."""
    pairs = reads = 0
    w = c["window"]
    for n, length in zip(*_lengths(c)):
        first = length - n
        for p in (range(first, length) if w else ()):
            pairs += min(w, p + 1)
        if not w:
            pairs += n * first + n * (n + 1) // 2
        reads += min(length, n + w - 1) if w else length
    return pairs, reads


def work(c):
    sz = _SZ[c["dtype"]]
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * sz + 8 * c["tokens"], "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    new, lens = _lengths(c)
    if c["op"] == "append":
        row = c["kv_heads"] * c["dim"]
        back = sum(length - (length - n) // c["page"] * c["page"] for n, length in zip(new, lens))
        n = sum(new)
        # the new keys and values in, their bytes out; then the pages they touch read and given back
        return {"bytes": 2 * row * (n * (sz + 1) + back * (1 + (2 if c["rot"] else sz))), "flops": 2 * row * (2 * n + back + (3 * n if c["rot"] else 0))}
    pairs, reads = _pairs(c)
    n = sum(new)
    by = 2 * reads * c["kv_heads"] * c["dim"] + 2 * n * c["q_heads"] * c["dim"] * sz + 4 * n * c["q_heads"]
    return {"bytes": by + 12 * sum(-(-x // c["page"]) for x in lens), "flops": 4 * pairs * c["q_heads"] * c["dim"]}


# ---------------------------------------------------------------------------------------------
# inputs


def _rope_config(c):
    if c["op"] == "rope":
        return dict(rot_dim=c["rot"], base=10000.0, layout=c["layout"], scaling=c["scaling"], factor=c["factor"],
                    original_max_position=max(16, int(c["max_pos"] / c["factor"])))
    if not c["rot"]:
        return None
    return dict(rot_dim=c["rot"], base=1000000.0, layout="half", scaling="none", factor=1.0, original_max_position=4096)


def _inv_freq(r):
    """Rotary frequencies in 64 bits (host), and the factor on the result."""
    n = r["rot_dim"] // 2
    d, base, f = r["rot_dim"], r["base"], r["factor"]
    if r["scaling"] == "ntk":
        base = base * f ** (d / (d - 2))
    inv = [base ** (-2.0 * i / d) for i in range(n)]
    if r["scaling"] == "linear":
        return [x / f for x in inv], 1.0
    if r["scaling"] == "yarn":
        def at(turns):
            return d * math.log(r["original_max_position"] / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(0, math.floor(at(32.0))), min(d - 1, math.ceil(at(1.0)))
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(n)]
        return [x / f * t + x * (1 - t) for x, t in zip(inv, ramp)], 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _scale_of(amax):
    """The least power of two 2^e, e >= -126, with amax <= 448 * 2^e (fp32)."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -126)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(amax), e)


def _pool(g, n_pages, heads, page, dim, spread):
    """A cache pool as a serving loop has it: values around 1, a few strong channels (`spread`), quantised by the rule above."""
    pages = torch.empty((n_pages, heads, page, dim), dtype=torch.float8_e4m3fn, device=_DEV)
    scales = torch.empty((n_pages, heads), dtype=torch.float32, device=_DEV)
    ch = 1.0 + spread * (torch.rand((heads, 1, dim), device=_DEV, generator=g) > 0.95)
    step = max(1, (1 << 27) // (heads * page * dim))
    for a in range(0, n_pages, step):
        b = min(n_pages, a + step)
        x = torch.randn((b - a, heads, page, dim), device=_DEV, generator=g) * ch
        s = _scale_of(x.abs().amax(dim=(2, 3)))
        pages[a:b] = (x / s[:, :, None, None]).to(torch.float8_e4m3fn)
        scales[a:b] = s
    return pages, scales


def _inputs(c, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    dt = _DT[c["dtype"]]
    st = {"case": c}
    r = _rope_config(c)
    if r is not None:
        inv, amp = _inv_freq(r)
        st["rope"], st["amp"] = r, amp
        # turns per position as a 64-bit fraction: position * fraction wraps to the turn's own fraction
        fx = [int(round(x / (2 * math.pi) * 2 ** 64)) for x in inv]
        st["turns"] = torch.tensor([x - (1 << 64) if x >= 1 << 63 else x for x in fx], dtype=torch.int64, device=_DEV)
    if c["op"] == "rope":
        st["x"] = torch.randn((c["tokens"], c["heads"], c["dim"]), device=_DEV, generator=g).to(dt)
        st["pos"] = torch.randint(0, c["max_pos"], (c["tokens"],), device=_DEV, generator=g, dtype=torch.int32)
        return st
    new, lens = _lengths(c)
    page, heads, dim = c["page"], c["kv_heads"], c["dim"]
    need = [-(-x // page) for x in lens]
    n_pages = sum(need) + 3
    perm = torch.randperm(n_pages, device=_DEV, generator=g).to(torch.int32).tolist()
    table = torch.full((c["seqs"], max(need)), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = torch.tensor(perm[at:at + k], dtype=torch.int32)
        at += k
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    st["table"] = table.to(_DEV)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=_DEV)
    st["offsets"] = torch.tensor(offsets, dtype=torch.int64, device=_DEV)
    st["n_tokens"], st["max_new"], st["max_len"] = offsets[-1], max(new), max(lens)
    st["k_pages"], st["k_scales"] = _pool(g, n_pages, heads, page, dim, 6.0)
    st["v_pages"], st["v_scales"] = _pool(g, n_pages, heads, page, dim, 1.0)
    # what lies behind a sequence's last token is whatever the memory held: NaN bytes among it
    for s, x in enumerate(lens):
        if x % page:
            p = int(table[s, need[s] - 1])
            st["k_pages"].view(torch.uint8)[p, :, x % page:] = 0x7F
            st["v_pages"].view(torch.uint8)[p, :, x % page:] = 0x7F
    if c["op"] == "append":
        n = st["n_tokens"]
        st["k"] = (torch.randn((n, heads, dim), device=_DEV, generator=g) * 1.5).to(dt)
        st["v"] = torch.randn((n, heads, dim), device=_DEV, generator=g).to(dt)
        # the pages that the new tokens touch, from the first page's start
        back = [x - (x - k) // page * page for k, x in zip(new, lens)]
        off = [0]
        for b in back:
            off.append(off[-1] + b)
        st["back_offsets"] = torch.tensor(off, dtype=torch.int64, device=_DEV)
        st["n_back"], st["max_back"] = off[-1], max(back)
    else:
        st["q"] = torch.randn((st["n_tokens"], c["q_heads"], dim), device=_DEV, generator=g).to(dt)
    return st


def prepare(c, seed):
    st = _inputs(c, seed)
    if own:
        pkg = str(Path(__file__).resolve().parent.parent / "sixi-asi_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from sixi_smp.kv_cache import KvBatch, KvCache, Rope

        if "rope" in st:
            st["h_rope"] = Rope(**st["rope"])
        if c["op"] != "rope":
            st["cache"] = KvCache(st["k_pages"].shape[0], c["page"], c["kv_heads"], c["dim"], k_pages=st["k_pages"],
                                  v_pages=st["v_pages"], k_scales=st["k_scales"], v_scales=st["v_scales"])
            st["batch"] = KvBatch(st["table"], st["offsets"], st["lens"], st["n_tokens"], st["max_new"])
        if c["op"] == "append":
            st["back"] = KvBatch(st["table"], st["back_offsets"], st["lens"], st["n_back"], st["max_back"])
    return st


# ---------------------------------------------------------------------------------------------
# one pass


def run(st):
    c = st["case"]
    if not own:
        return {"rope": _plain_rope_case, "append": _plain_append, "attend": _plain_attend}[c["op"]](st)
    if c["op"] == "rope":
        return st["h_rope"].apply(st["x"], st["pos"], inverse=c["inverse"])
    if c["op"] == "append":
        status = st["cache"].append(st["k"], st["v"], st["batch"], rope=st.get("h_rope"))
        k, v = st["cache"].read(st["back"], dtype=_read_type(c))
        return {"k": k, "v": v, "status": status}
    out, lse, status = st["cache"].attend(st["q"], st["batch"], window=c["window"], rope=st.get("h_rope"))
    return {"out": out, "lse": lse, "status": status}


def _plain_rotate(st, x, pos, inverse):
    """x [n, heads, dim] in 32 bits, turned by its positions [n]."""
    r = st["rope"]
    rot = r["rot_dim"]
    frac = pos.to(torch.int64)[:, None] * st["turns"][None, :]  # wraps at whole turns
    angle = frac.to(torch.float32) * (2.0 * math.pi / 2.0 ** 64)
    cos = (torch.cos(angle) * st["amp"])[:, None, :]
    sin = (torch.sin(angle) * (-st["amp"] if inverse else st["amp"]))[:, None, :]
    if r["layout"] == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    ya, yb = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([ya, yb], -1) if r["layout"] == "half" else torch.stack([ya, yb], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_rope_case(st):
    x = st["x"]
    return _plain_rotate(st, x.float(), st["pos"], st["case"]["inverse"]).to(x.dtype)


def _token_places(st, offsets, n):
    """(sequence, position) of each of the n tokens of a batch."""
    i = torch.arange(n, device=_DEV)
    seq = torch.searchsorted(offsets[1:], i, right=True)
    return seq, st["lens"].long()[seq] - (offsets[seq + 1] - i)


def _plain_write(pages, scales, x, page_id, slot, first, has_old):
    """Tokens x [n, heads, dim] (32 bits) into their pages; first, has_old [seqs]: each sequence's first
    touched page, and whether it holds older tokens."""
    n, heads, _ = x.shape
    amax = torch.zeros_like(scales)
    amax.scatter_reduce_(0, page_id[:, None].expand(n, heads), x.abs().amax(-1), "amax")
    new = _scale_of(amax)
    old, s = scales[first], new[first]
    s = torch.where(has_old[:, None], torch.maximum(old, s), s)
    keep = torch.where(has_old[:, None], old / s, torch.ones_like(s))
    new[first] = s
    held = (pages[first].view(torch.float8_e4m3fn).float() * keep[:, :, None, None]).to(torch.float8_e4m3fn)
    pages[first] = held.view(torch.uint8)
    at = new[page_id]
    pages[page_id, :, slot] = (x / at[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[page_id] = at


def _read_type(c):
    """What a case reads the cache back in. Every cached value is exact in bf16, which is what a step on
    rotated keys takes on; fp32 where the keys came in fp32 and were kept as they are."""
    return torch.bfloat16 if c["rot"] else _DT[c["dtype"]]


def _plain_values(pages, scales, page_id, slot, dt):
    bits = pages.view(torch.uint8)[page_id, :, slot].view(torch.float8_e4m3fn)
    return (bits.float() * scales[page_id][:, :, None]).to(dt)


def _plain_append(st):
    c = st["case"]
    page = c["page"]
    n = st["n_tokens"]
    seq, pos = _token_places(st, st["offsets"], n)
    start = st["lens"].long() - (st["offsets"][1:] - st["offsets"][:-1])
    page_id, slot = st["table"].long()[seq, pos // page], pos % page
    first, has_old = st["table"].long().gather(1, (start // page)[:, None])[:, 0], start % page > 0
    k, v = st["k"].float(), st["v"].float()
    if "rope" in st:
        k = _plain_rotate(st, k, pos, False)
    _plain_write(st["k_pages"].view(torch.uint8), st["k_scales"], k, page_id, slot, first, has_old)
    _plain_write(st["v_pages"].view(torch.uint8), st["v_scales"], v, page_id, slot, first, has_old)
    seq, pos = _token_places(st, st["back_offsets"], st["n_back"])
    page_id, slot = st["table"].long()[seq, pos // page], pos % page
    dt = _read_type(c)
    return {"k": _plain_values(st["k_pages"], st["k_scales"], page_id, slot, dt),
            "v": _plain_values(st["v_pages"], st["v_scales"], page_id, slot, dt),
            "status": torch.zeros(c["seqs"], dtype=torch.int32, device=_DEV)}


def _plain_attend(st):
    c = st["case"]
    page, heads, dim, group = c["page"], c["kv_heads"], c["dim"], c["q_heads"] // c["kv_heads"]
    b, length, rows = c["seqs"], st["table"].shape[1] * page, st["max_new"]
    lens = st["lens"].long()
    seq, pos = _token_places(st, st["offsets"], st["n_tokens"])
    q = st["q"].float()
    if "rope" in st:
        q = _plain_rotate(st, q, pos, False).to(st["q"].dtype).float()
    row = torch.arange(st["n_tokens"], device=_DEV) - st["offsets"][seq]
    qp = torch.zeros((b, rows, c["q_heads"], dim), device=_DEV)
    qp[seq, row] = q
    pp = torch.full((b, rows), -1, dtype=torch.int64, device=_DEV)
    pp[seq, row] = pos
    ids = st["table"].long().clamp(min=0)
    t = torch.arange(length, device=_DEV)
    inside = (t[None, :] < lens[:, None])[:, None, :, None]

    def cached(pages, scales):
        x = pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()  # [b, pages, heads, page, dim]
        x *= scales[ids][..., None, None]
        return torch.where(inside, x.transpose(1, 2).reshape(b, heads, length, dim), 0.0)

    k, v = cached(st["k_pages"], st["k_scales"]), cached(st["v_pages"], st["v_scales"])
    qh = qp.reshape(b, rows, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(b, heads, group * rows, dim)
    s = (qh @ k.transpose(2, 3)).mul_(dim ** -0.5).view(b, heads, group, rows, length)
    ok = t[None, None, :] <= pp[:, :, None]
    if c["window"]:
        ok &= t[None, None, :] > pp[:, :, None] - c["window"]
    s.masked_fill_(~ok[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, heads, group * rows, length) @ v).view(b, heads, group, rows, dim) / total.clamp(min=1e-38)
    lse = (m + total.log())[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(b, rows, c["q_heads"], dim)[seq, row]
    lse = lse.permute(0, 3, 1, 2).reshape(b, rows, c["q_heads"])[seq, row]
    return {"out": o.to(st["q"].dtype), "lse": lse, "status": torch.zeros(b, dtype=torch.int32, device=_DEV)}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits


def _exact_rotate(r, x, pos, inverse):
    inv, amp = _inv_freq(r)
    rot = r["rot_dim"]
    angle = pos.double()[:, None] * torch.tensor(inv, dtype=torch.float64, device=x.device)
    z = torch.polar(torch.full_like(angle, amp), -angle if inverse else angle)[:, None, :]
    y = x.clone()
    if r["layout"] == "half":
        w = torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2: rot].contiguous()) * z
        y[..., : rot // 2], y[..., rot // 2: rot] = w.real, w.imag
    else:
        w = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * z
        y[..., 0:rot:2], y[..., 1:rot:2] = w.real, w.imag
    return y


def _exact_e4m3(x):
    """x (64 bits, |x| <= 448) rounded to e4m3, ties to even: 4 significant bits, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_pages(pages, scales, x, start, page, row):
    """Values of one sequence's touched pages after writing x [n, heads, dim] at positions from `start`."""
    out = []
    end = start + x.shape[0]
    for first in range(start // page * page, end, page):
        pid = int(row[first // page])
        lo, hi = max(first, start), min(first + page, end)
        new = x[lo - start:hi - start]
        amax = new.abs().amax(dim=(0, 2))
        m, e = torch.frexp(amax)
        e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -126)).clamp(min=-126)
        s = torch.ldexp(torch.ones_like(amax), e)
        if lo > first:
            before = scales[pid].double()
            s = torch.maximum(s, before)
            held = pages[pid, :, : lo - first].double() * (before / s)[:, None, None]
            out.append((_exact_e4m3(held) * s[:, None, None]).transpose(0, 1))
        out.append(_exact_e4m3(new / s[None, :, None]) * s[None, :, None])
    return torch.cat(out)


def exact(c, seed):
    st = _inputs(c, seed)
    if c["op"] == "rope":
        return _exact_rotate(st["rope"], st["x"].double(), st["pos"], c["inverse"])
    new, lens = _lengths(c)
    page, heads, dim = c["page"], c["kv_heads"], c["dim"]
    off = st["offsets"].tolist()
    table = st["table"].cpu()
    if c["op"] == "append":
        ks, vs = [], []
        for s, (n, length) in enumerate(zip(new, lens)):
            k, v = st["k"][off[s]:off[s + 1]].double(), st["v"][off[s]:off[s + 1]].double()
            pos = torch.arange(length - n, length, device=_DEV)
            if "rope" in st:
                k = _exact_rotate(st["rope"], k, pos, False)
            ks.append(_exact_pages(st["k_pages"], st["k_scales"], k, length - n, page, table[s]))
            vs.append(_exact_pages(st["v_pages"], st["v_scales"], v, length - n, page, table[s]))
        return {"k": torch.cat(ks), "v": torch.cat(vs), "status": None}
    group, w = c["q_heads"] // heads, c["window"]
    outs, lses = [], []
    for s, (n, length) in enumerate(zip(new, lens)):
        ids = table[s, : -(-length // page)].long().to(_DEV)
        pos = torch.arange(length - n, length, device=_DEV)
        q = st["q"][off[s]:off[s + 1]].double()
        if "rope" in st:
            # rounded to the queries' type after the turn, as the operator is defined
            q = _exact_rotate(st["rope"], q, pos, False).to(st["q"].dtype).double()
        o = torch.empty((n, c["q_heads"], dim), dtype=torch.float64, device=_DEV)
        lse = torch.empty((n, c["q_heads"]), dtype=torch.float64, device=_DEV)
        t = torch.arange(length, device=_DEV)
        ok = t[None, :] <= pos[:, None]
        if w:
            ok &= t[None, :] > pos[:, None] - w
        for h in range(heads):
            k, v = ((pages.view(torch.uint8)[ids, h].view(torch.float8_e4m3fn).double() * scales[ids, h].double()[:, None, None]).reshape(-1, dim)[:length]
                    for pages, scales in ((st["k_pages"], st["k_scales"]), (st["v_pages"], st["v_scales"])))
            for j in range(h * group, (h + 1) * group):
                z = (q[:, j] @ k.T) / math.sqrt(dim)
                z = z.masked_fill(~ok, -math.inf)
                lse[:, j] = torch.logsumexp(z, -1)
                o[:, j] = torch.softmax(z, -1) @ v
        outs.append(o)
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses), "status": None}
