"""The 8-bit paged key/value cache (include/sixi_kv.h) over torch CUDA tensors.

A serving step on a batch of streams, before the sampler or the verifier sees its logits:

    rope = Rope(rot_dim=128, base=1e6)
    cache = KvCache(n_pages, page_size=64, n_kv_heads=8, head_dim=128)
    batch = KvBatch(page_table, offsets, lens, n_tokens, max_new)
    cache.append(k, v, batch, rope=rope)                 # the new tokens' keys and values
    out, lse, status = cache.attend(q, batch, rope=rope)  # their queries over all cached tokens

`batch` names each sequence's last offsets[s + 1] - offsets[s] positions: one token a stream for a
decode step, 1 + k for speculative verification, a chunk of a prompt. After the verifier has accepted
a of k drafts, lens for the next batch continues from lens - k + a. A rejected draft whose keys or values were
the largest of its page leaves the page's scale raised, and its older tokens rounded at that.

Calls run on the current stream, or on `stream`: what they allocate then belongs to that stream, and what
they are given stays as it is until that stream is through with it. Which stream waits for which is the
caller's to say (events).
"""

from __future__ import annotations

import ctypes
import threading

from . import BF16, F32, _check, _lib, _ptr, on_stream

_P = ctypes.c_void_p
ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
ATTEND_ALL = 1  # SIXI_KV_ATTEND_ALL


class KvConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("n_pages", "page_size", "n_kv_heads", "head_dim", "max_seqs", "reserved")]


class KvTensor(ctypes.Structure):
    _fields_ = [("data", _P), ("dtype", ctypes.c_uint32), ("n_heads", ctypes.c_uint32),
                ("token_stride", ctypes.c_uint64), ("head_stride", ctypes.c_uint64)]


class KvBatchStruct(ctypes.Structure):
    _fields_ = [("page_table", _P), ("table_stride", ctypes.c_uint64), ("offsets", _P), ("lens", _P),
                ("n_seqs", ctypes.c_uint32), ("max_pages", ctypes.c_uint32), ("n_tokens", ctypes.c_uint32),
                ("max_new", ctypes.c_uint32)]


class RopeConfig(ctypes.Structure):
    _fields_ = [("rot_dim", ctypes.c_uint32), ("layout", ctypes.c_uint32), ("scaling", ctypes.c_uint32),
                ("original_max_position", ctypes.c_uint32), ("base", ctypes.c_double), ("factor", ctypes.c_double),
                ("beta_fast", ctypes.c_double), ("beta_slow", ctypes.c_double)]


def _dev_index(device) -> int:
    import torch

    if device is None:
        return torch.cuda.current_device()
    d = torch.device(device) if not isinstance(device, int) else torch.device("cuda", device)
    return d.index if d.index is not None else torch.cuda.current_device()


class _Records(threading.local):
    """The records that a call passes, one set a thread: the interpreter lock is dropped while the library reads them."""

    def __init__(self):
        self.views = (KvTensor(), KvTensor())
        self.at = tuple(ctypes.addressof(v) for v in self.views)


class _Caller:
    """What the calls of one handle share: a step makes one or two of them a layer, so the records that they pass
    are made once (a thread) and filled in place, and the stream is asked for without making a torch object of it."""

    def __init__(self, device: int):
        import torch

        self.torch, self.device, self.dev = torch, device, torch.device("cuda", device)
        self.dtypes = {torch.float32: F32, torch.bfloat16: BF16}
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.records = _Records()

    def stream(self, stream) -> int:
        if stream is not None:
            return int(stream.cuda_stream)
        if self.raw_stream is not None:
            return self.raw_stream(self.device)
        return int(self.torch.cuda.current_stream(self.device).cuda_stream)

    def here(self, t, what: str) -> None:
        """Refuses a tensor that does not lie on the handle's device: its address would be read or written there."""
        if not t.is_cuda or t.get_device() != self.device:
            raise ValueError(f"{what}: on {t.device}, not cuda:{self.device}")

    def view(self, i: int, t, tokens: int, dim: int, what: str, written: bool = False) -> int:
        """Record i filled with t [tokens, heads, dim] (unit stride along dim); its address."""
        dt = self.dtypes.get(t.dtype)
        shape = t.shape
        if dt is None or len(shape) != 3 or shape[0] != tokens or shape[2] != dim:
            raise ValueError(f"{what}: fp32 or bf16 [{tokens}, heads, {dim}] expected, got {t.dtype} {tuple(shape)}")
        self.here(t, what)
        stride = t.stride()
        if stride[2] != 1:
            raise ValueError(f"{what}: the last dimension must have unit stride")
        if written and ((stride[0] == 0 and shape[0] > 1) or (stride[1] == 0 and shape[1] > 1)):
            raise ValueError(f"{what}: rows that share their memory cannot be written")
        r = self.records
        v = r.views[i]
        v.data, v.dtype, v.n_heads, v.token_stride, v.head_stride = t.data_ptr(), dt, shape[1], stride[0], stride[1]
        return r.at[i]


def _rope_handle(rope):
    """The rotation that a call passes; a closed one is refused, since no handle means no rotation."""
    if rope is None:
        return None
    if not rope.h:
        raise ValueError("rope: closed")
    return rope.h


class Rope:
    """Rotary frequencies on one device (sixi_kv_rope_create). layout "half" or "interleaved"; scaling
    "none", "linear", "ntk" or "yarn" (factor; yarn also original_max_position and the betas). Calls only read
    it, so several threads and streams may use one at a time."""

    def __init__(self, rot_dim: int, base: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_max_position: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device=None):
        if layout not in ROPE_LAYOUTS or scaling not in ROPE_SCALINGS:
            raise ValueError(f"unknown rotary layout {layout!r} or scaling {scaling!r}")
        for what, v in (("rot_dim", rot_dim), ("original_max_position", original_max_position)):
            if not 0 <= v < 2 ** 32:  # (ctypes would take its low 32 bits)
                raise ValueError(f"{what}: {v} does not fit 32 bits")
        self.h = None
        self.device = _dev_index(device)
        self.call = _Caller(self.device)
        self.rot_dim = rot_dim
        c = RopeConfig(rot_dim, ROPE_LAYOUTS[layout], ROPE_SCALINGS[scaling], original_max_position, base, factor,
                       beta_fast, beta_slow)
        h = _P()
        _check("sixi_kv_rope_create", _lib().sixi_kv_rope_create(self.device, ctypes.byref(c), ctypes.byref(h)))
        self.h = h

    def close(self) -> None:
        if self.h:
            _lib().sixi_kv_rope_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @on_stream
    def apply(self, x, positions, inverse: bool = False, out=None, stream=None):
        """x [tokens, heads, dim] turned by positions [tokens] (int32); inverse turns back (the gradient).
        out may be x."""
        c, n, dim = self.call, x.shape[0], x.shape[-1]
        if positions.dtype != c.torch.int32 or positions.shape != (n,) or not positions.is_contiguous():
            raise ValueError("positions: contiguous int32 [tokens] expected")
        c.here(positions, "positions")
        if out is None:
            out = c.torch.empty_like(x)
        elif out.shape != x.shape:
            raise ValueError(f"out: {tuple(x.shape)} expected, got {tuple(out.shape)}")
        st = _lib().sixi_kv_rope_apply(self.h, c.view(0, x, n, dim, "x"), positions.data_ptr(), n, dim, 1 if inverse else 0,
                                       c.view(1, out, n, dim, "out", True), c.stream(stream))
        _check("sixi_kv_rope_apply", st)
        return out


class KvBatch:
    """The positions a call works on (sixi_kv_batch): page_table int32 [seqs, max_pages], offsets int64
    [seqs + 1], lens int32 [seqs] (tensors of the cache's device, kept alive here), and on the host the total
    number of tokens and the most of one sequence."""

    def __init__(self, page_table, offsets, lens, n_tokens: int, max_new: int):
        import torch

        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1:
            raise ValueError("page_table: int32 [seqs, max_pages] with unit stride along pages expected")
        n = page_table.shape[0]
        if offsets.dtype != torch.int64 or offsets.shape != (n + 1,) or not offsets.is_contiguous():
            raise ValueError(f"offsets: contiguous int64 [{n + 1}] expected")
        if lens.dtype != torch.int32 or lens.shape != (n,) or not lens.is_contiguous():
            raise ValueError(f"lens: contiguous int32 [{n}] expected")
        if not page_table.is_cuda or not (page_table.device == offsets.device == lens.device):
            raise ValueError("page_table, offsets, lens: one CUDA device expected, got "
                             f"{page_table.device}, {offsets.device}, {lens.device}")
        self.page_table, self.offsets, self.lens = page_table, offsets, lens
        self.tensors = (page_table, offsets, lens)
        self.n_seqs, self.n_tokens, self.max_new = n, int(n_tokens), int(max_new)
        self.struct = KvBatchStruct(page_table.data_ptr(), page_table.stride(0), offsets.data_ptr(), lens.data_ptr(), n,
                                    page_table.shape[1], self.n_tokens, self.max_new)
        self.at = ctypes.addressof(self.struct)


class KvCache:
    """A cache on one device (sixi_kv_create). The pages are torch tensors: uint8 or float8_e4m3fn
    [n_pages, n_kv_heads, page_size, head_dim] and fp32 scales [n_pages, n_kv_heads], allocated here
    unless given. Its calls share a workspace: the caller puts them in order (one stream, or streams
    ordered by events)."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, k_pages=None, v_pages=None,
                 k_scales=None, v_scales=None, max_seqs: int = 4096, device=None):
        import torch

        self.h = None
        given = next((t for t in (k_pages, v_pages, k_scales, v_scales) if t is not None), None)
        self.device = _dev_index(given.device if device is None and given is not None else device)
        self.call = _Caller(self.device)
        dev = self.call.dev
        shape = (n_pages, n_kv_heads, page_size, head_dim)

        def buffer(t, shape, dtypes, what):
            if t is None:
                return torch.empty(shape, dtype=dtypes[0], device=dev)
            if tuple(t.shape) != shape or t.dtype not in dtypes or not t.is_contiguous() or t.device != dev:
                raise ValueError(f"{what}: contiguous {dtypes[0]} {shape} on {dev} expected, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
            return t

        by = (torch.uint8, torch.float8_e4m3fn)
        self.k_pages, self.v_pages = buffer(k_pages, shape, by, "k_pages"), buffer(v_pages, shape, by, "v_pages")
        self.k_scales = buffer(k_scales, shape[:2], (torch.float32,), "k_scales")
        self.v_scales = buffer(v_scales, shape[:2], (torch.float32,), "v_scales")
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = shape[0], page_size, n_kv_heads, head_dim
        c = KvConfig(n_pages, page_size, n_kv_heads, head_dim, max_seqs, 0)
        h = _P()
        st = _lib().sixi_kv_create(self.device, ctypes.byref(c), _ptr(self.k_pages), _ptr(self.v_pages),
                                   _ptr(self.k_scales), _ptr(self.v_scales), ctypes.byref(h))
        _check("sixi_kv_create", st)
        self.h = h

    def close(self) -> None:
        if self.h:
            _lib().sixi_kv_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _status(self, status, batch: KvBatch):
        """The call's status tensor, once the batch is known to lie on this device."""
        t = self.call.torch
        self.call.here(batch.page_table, "batch")
        if status is None:
            return t.empty(batch.n_seqs, dtype=t.int32, device=self.call.dev)
        if status.dtype != t.int32 or status.shape != (batch.n_seqs,) or not status.is_contiguous():
            raise ValueError(f"status: contiguous int32 [{batch.n_seqs}] expected")
        self.call.here(status, "status")
        return status

    @on_stream
    def append(self, k, v, batch: KvBatch, rope: Rope | None = None, status=None, stream=None):
        """Writes k, v [tokens, n_kv_heads, head_dim] at the batch's positions, the keys turned by rope.
        Returns the status of each sequence (int32, device)."""
        c, n, dim = self.call, batch.n_tokens, self.head_dim
        status = self._status(status, batch)
        st = _lib().sixi_kv_append(self.h, c.view(0, k, n, dim, "k"), c.view(1, v, n, dim, "v"), batch.at,
                                   _rope_handle(rope), status.data_ptr(), c.stream(stream))
        _check("sixi_kv_append", st)
        return status

    @on_stream
    def read(self, batch: KvBatch, dtype=None, k=None, v=None, status=None, stream=None):
        """The batch's positions as values: k, v [tokens, n_kv_heads, head_dim] (dtype bf16 or fp32)."""
        c, n, dim = self.call, batch.n_tokens, self.head_dim
        if k is None or v is None:
            dt = dtype or c.torch.bfloat16
            k = c.torch.empty((n, self.n_kv_heads, dim), dtype=dt, device=c.dev) if k is None else k
            v = c.torch.empty((n, self.n_kv_heads, dim), dtype=dt, device=c.dev) if v is None else v
        status = self._status(status, batch)
        st = _lib().sixi_kv_read(self.h, batch.at, c.view(0, k, n, dim, "k", True), c.view(1, v, n, dim, "v", True),
                                 status.data_ptr(), c.stream(stream))
        _check("sixi_kv_read", st)
        return k, v

    @on_stream
    def attend(self, q, batch: KvBatch, scale: float | None = None, window: int = 0, causal: bool = True,
               rope: Rope | None = None, out=None, lse=None, status=None, stream=None):
        """Attention of q [tokens, n_q_heads, head_dim] over the cache: (out like q, lse fp32 [tokens,
        n_q_heads], status int32 [seqs]). scale defaults to head_dim ** -0.5; window 0 is none."""
        c, n, dim = self.call, batch.n_tokens, self.head_dim
        if window < 0:
            raise ValueError(f"window: {window} is negative")
        if out is None:
            out = c.torch.empty_like(q)
        elif out.shape != q.shape:
            raise ValueError(f"out: {tuple(q.shape)} expected, got {tuple(out.shape)}")
        if lse is None:
            lse = c.torch.empty(q.shape[:2], dtype=c.torch.float32, device=c.dev)
        elif lse.dtype != c.torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous():
            raise ValueError(f"lse: contiguous fp32 {tuple(q.shape[:2])} expected")
        c.here(lse, "lse")
        status = self._status(status, batch)
        st = _lib().sixi_kv_attend(self.h, c.view(0, q, n, dim, "q"), batch.at,
                                   dim ** -0.5 if scale is None else scale, min(window, 0xFFFFFFFF),
                                   0 if causal else ATTEND_ALL, _rope_handle(rope), c.view(1, out, n, dim, "out", True),
                                   lse.data_ptr(), status.data_ptr(), c.stream(stream))
        _check("sixi_kv_attend", st)
        return out, lse, status
