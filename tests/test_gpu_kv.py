"""The 8-bit paged key/value cache on the GPU against its definition in 64 bits (kv_reference.py).

Tolerances, from the formulas (u = 2^-24 and b = 2^-8, the rounding units of fp32 and bf16):
  rotation  the angle is held to 2^-25 of a half turn after one rounding to fp32 (pi u), sine and cosine
            to 2 u, the products and their sum to 3 u: 10 u (|a| + |b|) amp in all, and b |y| for the
            rounding to bf16
  writing   none for unturned keys and values (bytes and scales equal); a turned key may fall to the
            neighbouring e4m3 value where the two sides' 64- and 32-bit angles straddle a midpoint:
            2^-3 of the value or the smallest step
  attention a score's error is at most (dim + 8) u times R, R the largest sum of scale |q| |k|; weights
            then err by a factor e^(2 err), their sum and the values' sum by another (length / 16 + 64) u
            (partial sums of 64 to 128 tokens); with bf16 queries the weights are rounded to 8
            significant bits (b) and the output to bf16 (b)
"""

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
import sixi_smp as S  # noqa: E402
from sixi_smp.kv_cache import KvBatch, KvCache, Rope  # noqa: E402

DEV = torch.device("cuda:0")
U, B = 2.0 ** -24, 2.0 ** -8
BF, F32 = torch.bfloat16, torch.float32


def host(t):
    return t.detach().to(torch.float64).cpu().numpy()


class World:
    """A cache on the GPU and its reference, with sequences' pages dealt at random."""

    def __init__(self, seed, lens, page, heads, dim, spare=2):
        self.rng = np.random.default_rng(seed)
        need = [max(1, -(-x // page)) for x in lens]
        n_pages = sum(need) + spare
        perm = self.rng.permutation(n_pages)
        self.table = np.full((len(lens), max(need)), -1, np.int32)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = perm[at:at + k]
            at += k
        self.lens, self.page, self.heads, self.dim = list(lens), page, heads, dim
        self.rk, self.rv = R.Cache(n_pages, heads, page, dim, self.rng), R.Cache(n_pages, heads, page, dim, self.rng)
        self.kv = KvCache(n_pages, page, heads, dim, device=0, max_seqs=max(16, len(lens)))
        self.push()

    def push(self):
        for t, a in ((self.kv.k_pages, self.rk.bytes), (self.kv.v_pages, self.rv.bytes),
                     (self.kv.k_scales, self.rk.scale), (self.kv.v_scales, self.rv.scale)):
            t.copy_(torch.from_numpy(a))

    def fill(self, upto=None):
        """Finite contents for every sequence, on both sides."""
        ch = 1 + 5 * (self.rng.random((1, self.heads, self.dim)) > 0.9)
        for s, n in enumerate(upto or self.lens):
            if n:
                self.rk.write(self.table[s], 0, self.rng.normal(size=(n, self.heads, self.dim)) * ch)
                self.rv.write(self.table[s], 0, self.rng.normal(size=(n, self.heads, self.dim)))
        self.push()
        return self

    def batch(self, new, lens=None, table=None):
        off = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        return KvBatch(torch.from_numpy(self.table if table is None else table).to(DEV), torch.from_numpy(off).to(DEV),
                       torch.tensor(self.lens if lens is None else lens, dtype=torch.int32, device=DEV), int(off[-1]),
                       max(new))

    def same_bytes(self, tol_turned=False):
        for t, r, sc, rs in ((self.kv.k_pages, self.rk.bytes, self.kv.k_scales, self.rk.scale),
                             (self.kv.v_pages, self.rv.bytes, self.kv.v_scales, self.rv.scale)):
            assert np.array_equal(sc.cpu().numpy(), rs)
            got = t.cpu().numpy()
            if tol_turned:
                a, b = R.E4M3[got], R.E4M3[r]
                assert np.array_equal(np.isnan(a), np.isnan(b))
                d = np.abs(a - b)
                assert np.nanmax(d - np.maximum(np.abs(b) / 8, 2.0 ** -9)) <= 0
                assert np.mean(d[~np.isnan(d)] != 0) < 1e-3
            else:
                assert np.array_equal(got, r)


# ---------------------------------------------------------------------------------------------
# rotary positions

ROPES = [
    dict(rot_dim=64, base=10000.0),
    dict(rot_dim=22, base=10000.0, layout="interleaved"),
    dict(rot_dim=80, base=500000.0, scaling="linear", factor=4.0),
    dict(rot_dim=128, base=10000.0, scaling="ntk", factor=8.0, layout="interleaved"),
    dict(rot_dim=96, base=10000.0, scaling="yarn", factor=16.0, original_max_position=4096),
    dict(rot_dim=2, base=10000.0),
]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("cfg", ROPES, ids=lambda c: f"{c['rot_dim']}{c.get('layout', 'half')[0]}-{c.get('scaling', 'none')}")
@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 128), (7, 3, 130), (300, 40, 160)])
def test_rope(cfg, dt, tokens, heads, dim):
    rng = np.random.default_rng(tokens + dim)
    x = torch.from_numpy(rng.normal(size=(tokens, heads, dim))).to(dt).to(DEV)
    pos = rng.integers(0, 2 ** 31 - 1, tokens).astype(np.int32)
    pos[0] = 0 if tokens > 1 else 123456
    r = Rope(device=0, **cfg)
    kw = {k: v for k, v in cfg.items() if k not in ("rot_dim", "layout")}
    freq, amp = R.inv_freq(cfg["rot_dim"], **kw)
    for inverse in (False, True):
        y = host(r.apply(x, torch.from_numpy(pos).to(DEV), inverse=inverse))
        ref = R.rotate(host(x), pos, freq, amp, cfg.get("layout", "half"), inverse)
        rot = cfg["rot_dim"]
        # the reference's own angle: position * f in 64 bits, off by up to 2^-53 of a 2^31 product
        tol = np.full_like(ref, (10 * U + 2.0 ** 31 * 2.0 ** -52) * amp) * 2 * np.abs(host(x)).max()
        tol[..., rot:] = 0.0
        if dt == BF:
            tol += B * np.abs(ref) * (np.arange(dim) < rot)
        assert np.all(np.abs(y - ref) <= tol)
    r.close()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_in_place_strided_and_its_gradient(layout):
    """Heads inside wider rows, out = x; the inverse call is the forward's gradient."""
    rng = np.random.default_rng(5)
    wide = torch.from_numpy(rng.normal(size=(50, 9, 100))).to(F32).to(DEV)
    x = wide[:, 1:8, 3:99]  # 96 elements at an odd offset: no 16-byte alignment
    before = wide.clone()
    pos = torch.arange(50, dtype=torch.int32, device=DEV) * 977
    r = Rope(64, layout=layout, scaling="yarn", factor=4.0, original_max_position=1024, device=0)
    freq, amp = R.inv_freq(64, scaling="yarn", factor=4.0, original_max_position=1024)
    ref = R.rotate(host(x), pos.cpu().numpy(), freq, amp, layout)
    assert r.apply(x, pos, out=x) is x
    assert np.abs(host(x) - ref).max() <= 20 * U * amp * np.abs(host(before)).max()
    assert torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, 8], before[:, 8])
    assert torch.equal(wide[:, :, :3], before[:, :, :3]) and torch.equal(wide[:, 1:8, 67:], before[:, 1:8, 67:])
    # gradient of sum(w * rope(x)): the inverse of w; against autograd of the formula, and a difference
    w = rng.normal(size=ref.shape)
    g = host(r.apply(torch.from_numpy(w).to(F32).to(DEV), pos, inverse=True))
    x64 = torch.from_numpy(host(before[:, 1:8, 3:99])).requires_grad_()
    ang = torch.from_numpy(pos.cpu().numpy().astype(np.float64)[:, None] * freq[None])
    c, s = amp * torch.cos(ang)[:, None], amp * torch.sin(ang)[:, None]
    a, b = (x64[..., :32], x64[..., 32:64]) if layout == "half" else (x64[..., 0:64:2], x64[..., 1:64:2])
    p, q = a * c - b * s, b * c + a * s
    y = torch.cat([torch.cat([p, q], -1) if layout == "half" else torch.stack([p, q], -1).flatten(-2), x64[..., 64:]], -1)
    (y * torch.from_numpy(w)).sum().backward()
    tol = 20 * U * amp * np.abs(w).max() * 2
    assert np.abs(g - x64.grad.numpy()).max() <= tol
    d = rng.normal(size=ref.shape)
    x0 = host(before[:, 1:8, 3:99])
    f = lambda z: float((R.rotate(z, pos.cpu().numpy(), freq, amp, layout) * w).sum())  # noqa: E731
    diff = (f(x0 + 1e-4 * d) - f(x0 - 1e-4 * d)) / 2e-4  # linear: only 64-bit rounding is lost
    assert abs(diff - float((g * d).sum())) <= tol * np.abs(d).sum() + 1e-6


# ---------------------------------------------------------------------------------------------
# writing and reading


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("page,heads,dim,old,new", [
    (16, 1, 16, [0, 15, 16, 31], [1, 1, 1, 1]),
    (16, 5, 96, [0, 7, 15, 16, 40, 3], [9, 1, 2, 33, 0, 16]),
    (32, 3, 80, [1, 64, 0], [70, 5, 1]),
    (64, 8, 128, [63, 10, 0, 200], [1, 200, 64, 3]),
    (128, 2, 256, [100, 5], [300, 2]),
    (128, 4, 64, [0], [1000]),
])
def test_append_bytes(dt, page, heads, dim, old, new):
    lens = [a + b for a, b in zip(old, new)]
    w = World(11, lens, page, heads, dim).fill(old)
    n = sum(new)
    # magnitudes over many binades, so that pages' scales grow, with zeros and subnormals among them
    mag = 2.0 ** w.rng.integers(-20, 12, size=(n, heads, 1))
    k = torch.from_numpy(w.rng.normal(size=(n, heads, dim)) * mag).to(dt)
    v = torch.from_numpy(w.rng.normal(size=(n, heads, dim))).to(dt)
    v[n // 2] = 0.0
    k[0, 0] = 1e-42 if dt == F32 else 0.0
    b = w.batch(new, lens)
    for _ in range(2):  # a second call with the same tokens changes nothing
        st = w.kv.append(k.to(DEV), v.to(DEV), b)
    at = 0
    for s, m in enumerate(new):
        if m:
            assert not w.rk.write(w.table[s], old[s], host(k[at:at + m]))
            assert not w.rv.write(w.table[s], old[s], host(v[at:at + m]))
        at += m
    w.same_bytes()
    assert st.tolist() == [0] * len(new)
    # reading back: everything up to the lengths, exact in fp32
    full = w.batch(lens, lens)
    kb, vb = w.kv.read(full, dtype=F32)
    at = 0
    for s, m in enumerate(lens):
        for h in range(heads):
            assert np.array_equal(host(kb[at:at + m, h]), w.rk.values(w.table[s], h, m).astype(np.float32))
            assert np.array_equal(host(vb[at:at + m, h]), w.rv.values(w.table[s], h, m).astype(np.float32))
        at += m


def test_append_scale_at_its_boundaries():
    """Magnitudes exactly at, and one ulp beyond, 448 * 2^e; the extremes of fp32."""
    vals = [448.0 * 2.0 ** e for e in (-126, -3, 0, 100)]
    vals += [float(np.nextafter(np.float32(v), np.float32(np.inf))) for v in vals] + [3.4e38, 1e-45, 0.0]
    w = World(3, [16] * len(vals), 16, 1, 16)
    x = np.zeros((len(vals), 1, 16), np.float32)
    x[:, 0, 0] = vals
    x[:, 0, 1] = -np.array(vals) / 3
    t = torch.from_numpy(x).to(DEV)
    st = w.kv.append(t, -t, w.batch([1] * len(vals), [1] * len(vals)))
    for s in range(len(vals)):
        w.rk.write(w.table[s], 0, x[s:s + 1])
        w.rv.write(w.table[s], 0, -x[s:s + 1])
    w.same_bytes()
    assert st.tolist() == [0] * len(vals)


def test_append_nan_and_inf_are_clamped_and_reported():
    lens = [20, 20, 20, 20]
    w = World(4, lens, 16, 2, 32).fill([10] * 4)
    x = w.rng.normal(size=(40, 2, 32)).astype(np.float32)
    x[3, 1, 5], x[12, 0, 0], x[13, 0, 1] = np.nan, np.inf, -np.inf
    y = x.copy()
    y[25] = np.nan  # a whole row of values
    y[35:40] = 0.0
    st = w.kv.append(torch.from_numpy(x).to(DEV), torch.from_numpy(y).to(DEV), w.batch([10] * 4))
    bad = []
    for s in range(4):
        a = w.rk.write(w.table[s], 10, x[10 * s:10 * s + 10])
        b = w.rv.write(w.table[s], 10, y[10 * s:10 * s + 10])
        bad.append(S.NUMERIC_NAN_OR_INF if a or b else 0)
    w.same_bytes()
    assert st.tolist() == bad == [16, 16, 16, 0]


def test_append_turned_keys_and_strided_inputs():
    old, new = [5, 0, 60], [4, 130, 10]
    lens = [a + b for a, b in zip(old, new)]
    w = World(6, lens, 64, 3, 96).fill(old)
    n = sum(new)
    wide = torch.from_numpy(w.rng.normal(size=(n, 7, 101))).to(F32).to(DEV)
    k, v = wide[:, 0:3, 2:98], wide[:, 4:7, 5:101]
    r = Rope(64, base=1e6, device=0)
    st = w.kv.append(k, v, w.batch(new), rope=r)
    freq, amp = R.inv_freq(64, base=1e6)
    at = 0
    for s, m in enumerate(new):
        pos = np.arange(old[s], lens[s])
        w.rk.write(w.table[s], old[s], R.rotate(host(k[at:at + m]), pos, freq, amp))
        w.rv.write(w.table[s], old[s], host(v[at:at + m]))
        at += m
    w.same_bytes(tol_turned=True)
    assert st.tolist() == [0, 0, 0]
    # aligned rows of the same values take the vector path: the same bytes
    kb = w.kv.k_pages.clone()
    w.kv.append(k.contiguous(), v.contiguous(), w.batch(new), rope=r)
    assert torch.equal(kb, w.kv.k_pages)


def test_append_and_read_report_what_does_not_fit():
    lens = [20, 20, 20, 20, 20, 0]
    w = World(8, lens, 16, 2, 32).fill([16, 16, 16, 16, 16, 0])
    n = 4
    x = torch.from_numpy(w.rng.normal(size=(5 * n, 2, 32))).to(F32).to(DEV)
    table = w.table.copy()
    table[1, 1] = -1
    table[2, 1] = w.rk.bytes.shape[0]
    before_k, before_v = w.kv.k_pages.clone(), w.kv.v_pages.clone()
    bad_lens = [20, 20, 20, 33, 3, 0]  # beyond the table; fewer than the new tokens
    b = w.batch([n] * 5 + [0], bad_lens, table)
    st = w.kv.append(x, x, b)
    assert st.tolist() == [0, 2, 2, 2, 2, 0]
    w.rk.write(w.table[0], 16, host(x[:4]))
    w.rv.write(w.table[0], 16, host(x[:4]))
    w.same_bytes()
    assert not torch.equal(before_k, w.kv.k_pages) and not torch.equal(before_v, w.kv.v_pages)
    k = torch.full((5 * n, 2, 32), 7.0, device=DEV)
    v = k.clone()
    status = torch.empty(6, dtype=torch.int32, device=DEV)
    w.kv.read(b, k=k, v=v, status=status)
    assert status.tolist() == [0, 2, 2, 2, 2, 0]
    assert np.array_equal(host(k[:4, 1]), w.rk.values(w.table[0], 1, 20)[16:].astype(np.float32))
    assert (k[4:12] == 0).all() and (v[4:12] == 0).all()  # bad ids
    assert (k[12:] == 7).all() and (v[12:] == 7).all()  # bad numbers


@pytest.mark.parametrize("offsets", [[0, 10, 5, 12], [0, 4, 8, 13], [-1, 4, 8, 12]])
def test_offsets_out_of_order_are_reported_by_every_sequence(offsets):
    w = World(10, [20, 20, 20], 16, 2, 32).fill()
    b = w.batch([4, 4, 4])
    x = torch.from_numpy(w.rng.normal(size=(12, 2, 32))).to(F32).to(DEV)
    want = host(w.kv.attend(x, b)[0])
    b.offsets.copy_(torch.tensor(offsets))
    y = torch.full_like(x, 7.0)
    for _ in range(2):  # (nothing is left behind that a later call would meet)
        assert w.kv.append(x, x, b).tolist() == [2, 2, 2]
        w.same_bytes()
        st = torch.zeros(3, dtype=torch.int32, device=DEV)
        w.kv.read(b, k=y, v=y.clone(), status=st)
        assert st.tolist() == [2, 2, 2] and (y == 7).all()
        for q in (x, x.to(BF)):
            assert w.kv.attend(q, b)[2].tolist() == [2, 2, 2]
    good = w.batch([4, 4, 4])
    out, _, st = w.kv.attend(x, good)
    assert st.tolist() == [0, 0, 0] and np.array_equal(host(out), want)
    assert w.kv.append(x, x, good).tolist() == [0, 0, 0]


def test_append_understated_max_new():
    """max_new picks a variant only."""
    w = World(9, [200], 64, 2, 128).fill([3])
    x = torch.from_numpy(w.rng.normal(size=(197, 2, 128))).to(BF)
    b = w.batch([197])
    b.struct.max_new = 1
    w.kv.append(x.to(DEV), x.to(DEV), b)
    w.rk.write(w.table[0], 3, host(x))
    w.rv.write(w.table[0], 3, host(x))
    w.same_bytes()


# ---------------------------------------------------------------------------------------------
# attention


def check_attend(w, new, hq, dt, window=0, causal=True, rope=None, rope_cfg=None, scale=None, q_scale=1.0, lens=None):
    lens = w.lens if lens is None else lens
    n = sum(new)
    q = torch.from_numpy(w.rng.normal(size=(n, hq, w.dim)) * q_scale).to(dt)
    b = w.batch(new, lens)
    out, lse, st = w.kv.attend(q.to(DEV), b, window=window, causal=causal, rope=rope, scale=scale)
    again, lse2, _ = w.kv.attend(q.to(DEV), b, window=window, causal=causal, rope=rope, scale=scale)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # the order of sums is fixed
    assert st.tolist() == [0] * len(new)
    sc = w.dim ** -0.5 if scale is None else scale
    at = 0
    for s, m in enumerate(new):
        qs = host(q[at:at + m])
        if rope is not None:
            freq, amp = R.inv_freq(**rope_cfg)
            qs = R.rotate(qs, np.arange(lens[s] - m, lens[s]), freq, amp)
        ro, rl, mag, reach = R.attend(w.rk, w.rv, w.table[s], lens[s], qs, sc, window, causal)
        err = (w.dim + 8) * U * reach
        if rope is not None:  # the turned query's rounding to its type
            err += (B if dt == BF else 12 * U) * reach
        weights = 2 * err + (lens[s] / 16 + 64) * U + (B if dt == BF else 0)
        tol = weights * mag * math.e + (B if dt == BF else 2 * U) * np.abs(ro) + 1e-30
        got, gl = host(out[at:at + m]), host(lse[at:at + m])
        assert np.all(np.abs(got - ro) <= tol), (s, np.abs(got - ro).max())
        empty = np.isinf(rl)
        assert np.array_equal(np.isneginf(gl), empty)
        assert np.all(got[empty] == 0)
        ltol = err + (lens[s] / 16 + 64) * U + 4 * U * np.abs(rl[~empty])
        assert np.all(np.abs(gl[~empty] - rl[~empty]) <= ltol)
        at += m


SHAPES = [  # page, key heads, group, dim, lens, new
    (16, 1, 1, 16, [1, 2, 16, 17, 33], [1, 1, 1, 1, 1]),
    (16, 2, 8, 64, [1, 127, 128, 129, 300], [1, 1, 1, 1, 1]),
    (64, 3, 7, 80, [33, 500, 64, 65], [1, 4, 2, 3]),
    (64, 2, 4, 128, [700], [1]),
    (32, 1, 8, 128, [400, 9, 130, 31], [9, 9, 5, 0]),
    (128, 1, 16, 128, [260, 1000], [5, 16]),
    (16, 1, 3, 96, [200, 90], [130, 90]),
    (64, 2, 2, 256, [300, 65, 129], [1, 40, 129]),
    (128, 1, 20, 192, [150, 129], [7, 1]),
    (64, 1, 5, 112, [513], [300]),
    (64, 1, 64, 64, [140], [2]),
    (16, 1, 130, 32, [37], [3]),
]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("page,heads,group,dim,lens,new", SHAPES)
def test_attend(dt, page, heads, group, dim, lens, new):
    w = World(21, lens, page, heads, dim).fill()
    check_attend(w, new, heads * group, dt)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("window", [1, 5, 64, 129, 10_000_000])
def test_attend_window(dt, window):
    w = World(22, [300, 70, 1, 129], 32, 2, 64).fill()
    check_attend(w, [150, 3, 1, 20], 6, dt, window=window)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_all_positions_and_scales(dt):
    w = World(23, [200, 40], 16, 1, 128).fill()
    check_attend(w, [100, 7], 4, dt, causal=False)
    check_attend(w, [100, 7], 4, dt, causal=False, window=30)
    check_attend(w, [100, 7], 4, dt, scale=0.0)
    check_attend(w, [100, 7], 4, dt, scale=-0.5)
    check_attend(w, [1, 7], 4, dt, q_scale=40.0)   # nearly one-hot weights
    check_attend(w, [1, 7], 4, dt, q_scale=1e-30)  # uniform weights


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_turns_queries(dt):
    w = World(24, [300, 70], 32, 2, 128).fill()
    cfg = dict(rot=96, base=1e5)
    r = Rope(96, base=1e5, device=0)
    check_attend(w, [9, 70], 8, dt, rope=r, rope_cfg=cfg)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_empty_rows(dt):
    """Sequences shorter than their new tokens, of length 0, without new tokens."""
    w = World(25, [3, 0, 0, 40, 130], 16, 2, 64).fill()
    check_attend(w, [8, 2, 0, 0, 140], 4, dt)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_long_split_over_the_grid(dt):
    w = World(26, [9000, 3, 2500], 128, 1, 64).fill()
    check_attend(w, [1, 1, 3], 2, dt)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_many_short_sequences(dt):
    lens = [int(x) for x in np.random.default_rng(5).integers(1, 40, 700)]
    w = World(27, lens, 16, 1, 32).fill()
    check_attend(w, [1] * 700, 2, dt)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_sink_and_a_long_tail(dt):
    """One token with nearly all the weight, thousands with the rest: the tail still counts."""
    n = 6000
    w = World(28, [n], 64, 1, 64)
    k = np.zeros((n, 1, 64))
    k[0, 0, 0] = 104.0
    v = np.ones((n, 1, 64))
    v[0] = 0.0
    v[1:, 0, 1] = 0.01
    w.rk.write(w.table[0], 0, k)
    w.rv.write(w.table[0], 0, v)
    w.push()
    q = torch.zeros((1, 1, 64), dtype=dt, device=DEV)
    q[0, 0, 0] = 1.0
    out, lse, _ = w.kv.attend(q, w.batch([1]), scale=0.125)
    ro, rl, mag, reach = R.attend(w.rk, w.rv, w.table[0], n, host(q), 0.125)
    assert np.all(np.abs(host(out) - ro) <= (2 * B) * mag + 1e-12)
    assert abs(float(lse[0, 0]) - rl[0, 0]) < 1e-4


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_pages_of_very_different_scales(dt):
    w = World(29, [96], 16, 1, 64)
    v = w.rng.normal(size=(96, 1, 64)) * np.repeat(2.0 ** np.array([0, -12, 9, -30, 3, 20]), 16)[:, None, None]
    k = w.rng.normal(size=(96, 1, 64)) * np.repeat(2.0 ** np.array([0, -3, 2, -30, 1, -9]), 16)[:, None, None]
    w.rk.write(w.table[0], 0, k)
    w.rv.write(w.table[0], 0, v)
    w.push()
    check_attend(w, [4], 2, dt)


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_nan_queries_stay_in_their_rows(dt):
    w = World(30, [100, 50], 16, 2, 64).fill()
    q = torch.from_numpy(w.rng.normal(size=(6, 8, 64))).to(dt).to(DEV)
    b = w.batch([4, 2])
    clean, lse0, _ = w.kv.attend(q, b)
    p = q.clone()
    p[1, 3, 7], p[2, 0, 0], p[5, 6, 63] = float("nan"), float("inf"), float("-inf")
    out, lse, st = w.kv.attend(p, b)
    bad = torch.zeros((6, 8), dtype=torch.bool, device=DEV)
    bad[1, 3] = bad[2, 0] = bad[5, 6] = True
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], lse0[~bad])
    assert st.tolist() == [0, 0]


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_strided_rows(dt):
    w = World(31, [100, 50], 16, 2, 64).fill()
    wide = torch.from_numpy(w.rng.normal(size=(12, 20, 70))).to(dt).to(DEV)
    q = wide[::2, 3:11, 1:65]
    b = w.batch([4, 2])
    want, lse0, _ = w.kv.attend(q.contiguous(), b)
    frame = torch.full((6, 10, 67), 5.0, dtype=dt, device=DEV)
    out, lse, _ = w.kv.attend(q, b, out=frame[:, 1:9, 2:66])
    assert torch.equal(out, want) and torch.equal(lse, lse0)
    assert (frame[:, 0] == 5).all() and (frame[:, 9] == 5).all() and (frame[:, :, :2] == 5).all() and (frame[:, :, 66:] == 5).all()


@pytest.mark.parametrize("dt", [BF, F32])
def test_attend_reports_what_does_not_fit(dt):
    lens = [100, 100, 100, 100]
    w = World(32, lens, 16, 1, 64).fill()
    q = torch.from_numpy(w.rng.normal(size=(4, 2, 64))).to(dt).to(DEV)
    good, _, _ = w.kv.attend(q, w.batch([1] * 4))
    t = w.table.copy()
    t[1, 3], t[2, 6] = w.rk.bytes.shape[0], -5
    out, _, st = w.kv.attend(q, w.batch([1] * 4, [100, 100, 100, 1000], t))
    assert st.tolist() == [0, 2, 2, 2]
    assert torch.equal(out[0], good[0])
    # ids that the window leaves out may be anything
    t = w.table.copy()
    t[:, 0], t[0, 1] = -7, 10 ** 9
    want, lse0, _ = w.kv.attend(q, w.batch([1] * 4), window=60)
    out, lse, st = w.kv.attend(q, w.batch([1] * 4, None, t), window=60)
    assert st.tolist() == [0] * 4 and torch.equal(out, want) and torch.equal(lse, lse0)


def test_attend_on_another_stream_and_in_a_graph():
    w = World(33, [400, 300], 64, 2, 128).fill()
    q = torch.from_numpy(w.rng.normal(size=(2, 8, 128))).to(BF).to(DEV)
    b = w.batch([1, 1])
    want, _, _ = w.kv.attend(q, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out, lse, st = w.kv.attend(q, b)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    o, l, s = torch.empty_like(out), torch.empty_like(lse), torch.empty_like(st)
    with torch.cuda.graph(g):
        w.kv.attend(q, b, out=o, lse=l, status=s)
    q.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    want, lse0, _ = w.kv.attend(q, b)
    assert torch.equal(o, want) and torch.equal(l, lse0)


def test_cache_beyond_4_gib():
    """Byte offsets that pass 32 bits: pages at the end of a 6 GB pool."""
    heads, page, dim = 8, 128, 256
    n_pages = 6 * 2 ** 30 // (heads * page * dim)
    kv = KvCache(n_pages, page, heads, dim, device=0, max_seqs=16)
    rng = np.random.default_rng(1)
    ids = np.array([[n_pages - 1, 0, n_pages // 2 + 1, n_pages - 2]], np.int32)
    rk, rv = R.Cache(4, heads, page, dim), R.Cache(4, heads, page, dim)
    x = rng.normal(size=(400, heads, dim)).astype(np.float32)
    b = KvBatch(torch.from_numpy(ids).to(DEV), torch.tensor([0, 400], device=DEV), torch.tensor([400], dtype=torch.int32, device=DEV),
                400, 400)
    t = torch.from_numpy(x).to(DEV)
    assert kv.append(t, -t, b).tolist() == [0]
    rk.write([0, 1, 2, 3], 0, x)
    rv.write([0, 1, 2, 3], 0, -x)
    k, v = kv.read(b, dtype=F32)
    for h in range(heads):
        assert np.array_equal(host(k[:, h]), rk.values([0, 1, 2, 3], h, 400).astype(np.float32))
        assert np.array_equal(host(v[:, h]), rv.values([0, 1, 2, 3], h, 400).astype(np.float32))
    b1 = KvBatch(b.page_table, torch.tensor([0, 1], device=DEV), b.lens, 1, 1)
    for dt in (F32, BF):
        q = torch.from_numpy(rng.normal(size=(1, 16, dim))).to(dt).to(DEV)
        out, _, _ = kv.attend(q, b1)
        ro, _, mag, reach = R.attend(rk, rv, [0, 1, 2, 3], 400, host(q), dim ** -0.5)
        tol = ((B if dt == BF else 0) + 2 * (dim + 8) * U * reach + 100 * U) * mag * math.e + B * np.abs(ro)
        assert np.all(np.abs(host(out) - ro) <= tol)


def test_python_checks():
    w = World(34, [20], 16, 2, 32).fill()
    b = w.batch([2])
    x = torch.zeros((2, 2, 32), device=DEV)
    for bad in (x[:1], x[:, :, :16], x.to(torch.float16), x.cpu(), x.transpose(1, 2)):
        with pytest.raises((ValueError, S.SixiError)):
            w.kv.append(bad, x, b)
    with pytest.raises(S.SixiError):  # three heads
        w.kv.append(torch.zeros((2, 3, 32), device=DEV), x, b)
    with pytest.raises(S.SixiError):  # mixed types
        w.kv.append(x, x.to(BF), b)
    with pytest.raises(S.SixiError):  # query heads that are no multiple
        w.kv.attend(torch.zeros((2, 3, 32), device=DEV), b)
    with pytest.raises(S.SixiError):
        w.kv.attend(torch.zeros((2, 4, 32), device=DEV), b, scale=float("nan"))
    with pytest.raises(S.SixiError):  # more turned elements than a head has
        w.kv.attend(torch.zeros((2, 4, 32), device=DEV), b, rope=Rope(64, device=0))
    with pytest.raises(ValueError):
        KvBatch(b.page_table.long(), b.offsets, b.lens, 2, 2)
    with pytest.raises(ValueError):
        Rope(64, layout="other", device=0)
    with pytest.raises(S.SixiError):
        KvCache(4, 24, 2, 32, device=0)


def test_tables_beyond_2_30_positions_are_refused():
    w = World(35, [20], 16, 2, 32).fill()
    b = w.batch([2])
    x = torch.zeros((2, 2, 32), device=DEV)
    b.struct.table_stride = 2 ** 28
    for pages in (2 ** 26 + 1, 2 ** 28):
        b.struct.max_pages = pages
        for call in (lambda: w.kv.append(x, x, b), lambda: w.kv.read(b, k=x, v=x), lambda: w.kv.attend(x, b)):
            with pytest.raises(S.SixiError):
                call()
