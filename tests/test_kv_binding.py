"""The cache's Python binding (sixi_smp.kv_cache) without a GPU: what it hands to the library, and what it refuses.

The library is a recorder, tensors are stand-ins that say where they lie: nothing is dereferenced."""

from __future__ import annotations

import contextlib
import ctypes
import math
import threading

import pytest
import torch

import sixi_smp
from sixi_smp import json_grammar, json_schema
from sixi_smp import kv_cache as K

I32, I64, F32, BF = torch.int32, torch.int64, torch.float32, torch.bfloat16


class Tensor:
    """What the binding asks a tensor for."""

    def __init__(self, shape, dtype, device="cuda:0", at=0x1000):
        self.shape, self.dtype, self.device, self.at = torch.Size(shape), dtype, torch.device(device), at
        self.is_cuda = self.device.type == "cuda"
        self.used_on = []

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        s = tuple(math.prod(self.shape[j + 1:]) for j in range(len(self.shape)))
        return s if i is None else s[i]

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device.index if self.is_cuda else -1

    def data_ptr(self):
        return self.at

    def numel(self):
        return math.prod(self.shape)

    def record_stream(self, stream):
        self.used_on.append(stream)


class Library:
    """Every entry point answers OK and is written down; `hook` sees the arguments first."""

    def __init__(self):
        self.calls, self.hook = [], None

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_create"):
                args[-1]._obj.value = 0x77
            if self.hook is not None:
                self.hook(name, args)
            self.calls.append(name)
            return 0

        return call


class Stream:
    def __init__(self, raw):
        self.cuda_stream, self.device = raw, torch.device("cuda:0")


MAIN, SIDE = Stream(7), Stream(8)
HANDLES = []


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    lib.current, lib.made = [MAIN], []
    for module in (K, sixi_smp, json_grammar, json_schema):
        monkeypatch.setattr(module, "_lib", lambda: lib)

    @contextlib.contextmanager
    def use(stream):
        lib.current.append(stream)
        yield
        lib.current.pop()

    def empty(shape, dtype=None, device=None):
        lib.made.append((lib.current[-1], Tensor((shape,) if isinstance(shape, int) else shape, dtype)))
        return lib.made[-1][1]

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: lib.current[-1])
    monkeypatch.setattr(torch.cuda, "stream", use)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch, "zeros", empty)
    monkeypatch.setattr(torch, "full", lambda shape, value, dtype=None, device=None: empty(shape, dtype))
    monkeypatch.setattr(torch, "empty_like", lambda t: empty(t.shape, t.dtype))
    yield lib
    for x in HANDLES:  # (the recorder's handles are nothing to the real library)
        x.h = None
    HANDLES.clear()


def make_cache(n_kv_heads=2, head_dim=32):
    pages = [Tensor((8, n_kv_heads, 16, head_dim), torch.uint8) for _ in range(2)]
    scales = [Tensor((8, n_kv_heads), F32) for _ in range(2)]
    HANDLES.append(K.KvCache(8, 16, n_kv_heads, head_dim, *pages, *scales, device=0))
    return HANDLES[-1]


def make_rope(rot_dim=32):
    HANDLES.append(K.Rope(rot_dim, device=0))
    return HANDLES[-1]


def batch(device="cuda:0", **where):
    at = {**dict.fromkeys(("page_table", "offsets", "lens"), device), **where}
    return K.KvBatch(Tensor((1, 4), I32, at["page_table"]), Tensor((2,), I64, at["offsets"]),
                     Tensor((1,), I32, at["lens"]), 3, 3)


# ---------------------------------------------------------------------------------------------
# where tensors lie: every address that reaches the library is one of the handle's device


@pytest.mark.parametrize("which", ["page_table", "offsets", "lens"])
@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
def test_batch_refuses_tensors_elsewhere(which, where):
    with pytest.raises(ValueError, match=which):
        batch(**{which: where})


def test_batch_refuses_host_tensors():
    """Real ones, as a caller would pass them."""
    with pytest.raises(ValueError, match="page_table"):
        K.KvBatch(torch.zeros((1, 4), dtype=I32), torch.tensor([0, 3]), torch.tensor([3], dtype=I32), 3, 3)


def calls_of(cache, b, status=None, lse=None):
    q, kv = Tensor((3, 4, 32), BF), Tensor((3, 2, 32), BF)
    status = status or Tensor((1,), I32)
    lse = lse or Tensor((3, 4), F32)
    return {"append": lambda: cache.append(kv, kv, b, status=status, stream=MAIN),
            "read": lambda: cache.read(b, k=kv, v=kv, status=status, stream=MAIN),
            "attend": lambda: cache.attend(q, b, out=q, lse=lse, status=status, stream=MAIN)}


@pytest.mark.parametrize("name", ["append", "read", "attend"])
def test_cache_refuses_a_batch_of_another_device(lib, name):
    cache = make_cache()
    with pytest.raises(ValueError, match="batch"):
        calls_of(cache, batch("cuda:1"))[name]()
    assert lib.calls == ["sixi_kv_create"]


@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
@pytest.mark.parametrize("name", ["append", "read", "attend"])
def test_cache_refuses_a_status_elsewhere(lib, name, where):
    cache = make_cache()
    with pytest.raises(ValueError, match="status"):
        calls_of(cache, batch(), status=Tensor((1,), I32, where))[name]()
    assert lib.calls == ["sixi_kv_create"]


@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
def test_attend_refuses_an_lse_elsewhere(lib, where):
    cache = make_cache()
    with pytest.raises(ValueError, match="lse"):
        calls_of(cache, batch(), lse=Tensor((3, 4), F32, where))["attend"]()
    assert lib.calls == ["sixi_kv_create"]


@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
def test_rope_refuses_positions_elsewhere(lib, where):
    rope = make_rope()
    x = Tensor((3, 2, 32), BF)
    with pytest.raises(ValueError, match="positions"):
        rope.apply(x, Tensor((3,), I32, where), out=x, stream=MAIN)
    assert lib.calls == ["sixi_kv_rope_create"]


def test_what_lies_on_the_device_is_passed_on(lib):
    cache = make_cache()
    for call in calls_of(cache, batch()).values():
        call()
    rope = make_rope()
    x = Tensor((3, 2, 32), BF)
    rope.apply(x, Tensor((3,), I32), out=x, stream=MAIN)
    assert lib.calls == ["sixi_kv_create", "sixi_kv_append", "sixi_kv_read", "sixi_kv_attend", "sixi_kv_rope_create",
                         "sixi_kv_rope_apply"]


# ---------------------------------------------------------------------------------------------
# threads: a call's records are its own while the library reads them


def test_two_threads_on_one_rope_keep_their_tensors(lib):
    """The interpreter may run another thread while a call is in the library: its records stay what they were."""
    rope = make_rope()
    meet, seen = threading.Barrier(2, timeout=20), {}

    def record(at):
        v = K.KvTensor.from_address(at)
        return v.data, v.token_stride, v.head_stride, v.n_heads

    def hook(name, args):
        meet.wait()  # both calls are inside the library
        before = record(args[1]), record(args[6])
        meet.wait()
        seen[before[0][0]] = before
        meet.wait()

    def work(i):
        x = Tensor((3, 2 + i, 32), BF, at=0x10000 * (i + 1))
        rope.apply(x, Tensor((3,), I32), out=Tensor((3, 2 + i, 32), BF, at=0x10000 * (i + 1) + 0x100), stream=MAIN)

    lib.hook = hook
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == {0x10000 * (i + 1): ((0x10000 * (i + 1), (2 + i) * 32, 32, 2 + i),
                                        (0x10000 * (i + 1) + 0x100, (2 + i) * 32, 32, 2 + i)) for i in range(2)}


# ---------------------------------------------------------------------------------------------
# streams: with `stream` given, nothing that the call touches is memory that another stream may still use, or be handed


def on_side(cache):
    q, k, v = Tensor((3, 4, 32), BF), Tensor((3, 2, 32), BF), Tensor((3, 2, 32), BF)
    b = batch()
    rope, pos = make_rope(), Tensor((3,), I32)
    own = [b.page_table, b.offsets, b.lens]
    return {"append": (lambda: cache.append(k, v, b, stream=SIDE), [k, v, *own]),
            "read": (lambda: cache.read(b, stream=SIDE), own),
            "attend": (lambda: cache.attend(q, b, stream=SIDE), [q, *own]),
            "apply": (lambda: rope.apply(q, pos, stream=SIDE), [q, pos])}


@pytest.mark.parametrize("name", ["append", "read", "attend", "apply"])
def test_a_named_stream_owns_what_the_call_makes(lib, name):
    call, given = on_side(make_cache())[name]
    result = call()
    assert lib.made and all(s is SIDE for s, _ in lib.made)
    assert all(t.used_on == [SIDE] for t in given)  # not handed out again before the side stream is through
    for t in result if isinstance(result, tuple) else (result,):
        assert t.used_on == [MAIN]  # the caller's stream reads it next
    assert lib.current == [MAIN]


def test_the_current_stream_costs_nothing(lib):
    cache = make_cache()
    q, b = Tensor((3, 4, 32), BF), batch()
    result = cache.attend(q, b, stream=MAIN)
    assert [s for s, _ in lib.made] == [MAIN] * 3
    assert not any(t.used_on for t in (*result, q, b.lens))


def test_a_stream_given_by_position(lib):
    cache = make_cache()
    k, v = Tensor((3, 2, 32), BF), Tensor((3, 2, 32), BF)
    cache.append(k, v, batch(), None, None, SIDE)
    assert [s for s, _ in lib.made] == [SIDE] and k.used_on == [SIDE]


# ---------------------------------------------------------------------------------------------
# arguments that would be taken for others


@pytest.mark.parametrize("name", ["append", "attend"])
def test_a_closed_rope_is_refused(lib, name):
    """Its handle is nothing, which the library takes for a call without a rotation."""
    cache, rope = make_cache(), make_rope()
    rope.close()
    q, kv, b = Tensor((3, 4, 32), BF), Tensor((3, 2, 32), BF), batch()
    with pytest.raises(ValueError, match="rope"):
        cache.append(kv, kv, b, rope=rope, stream=MAIN) if name == "append" else cache.attend(q, b, rope=rope, stream=MAIN)
    assert not {"sixi_kv_append", "sixi_kv_attend"} & set(lib.calls)


def test_windows_beyond_32_bits(lib):
    cache, seen = make_cache(), []
    lib.hook = lambda name, args: seen.append(ctypes.c_uint32(args[4]).value)
    q, b = Tensor((3, 4, 32), BF), batch()
    for window in (0, 5, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1):
        cache.attend(q, b, window=window, stream=MAIN)
    assert seen == [0, 5] + [2 ** 32 - 1] * 4
    for window in (-1, -2 ** 32 + 5):
        with pytest.raises(ValueError, match="window"):
            cache.attend(q, b, window=window, stream=MAIN)


@pytest.mark.parametrize("field", ["rot_dim", "original_max_position"])
@pytest.mark.parametrize("value", [-1, 2 ** 32 + 64])
def test_rope_numbers_beyond_32_bits_are_refused(lib, field, value):
    args = dict(rot_dim=64, scaling="yarn", factor=2.0, original_max_position=4096)
    with pytest.raises(ValueError, match=field):
        K.Rope(device=0, **{**args, field: value})


class Expanded(Tensor):
    """Every row of heads in the same place."""

    def stride(self, i=None):
        s = (0, 0, 1)
        return s if i is None else s[i]


@pytest.mark.parametrize("name", ["read", "attend", "apply"])
def test_outputs_whose_rows_share_their_place_are_refused(lib, name):
    cache, rope, b = make_cache(), make_rope(), batch()
    q, kv, one = Tensor((3, 4, 32), BF), Tensor((3, 2, 32), BF), Expanded((3, 2, 32), BF)
    calls = {"read": lambda: cache.read(b, k=kv, v=one, stream=MAIN),
             "attend": lambda: cache.attend(q, b, out=Expanded((3, 4, 32), BF), stream=MAIN),
             "apply": lambda: rope.apply(kv, Tensor((3,), I32), out=one, stream=MAIN)}
    with pytest.raises(ValueError, match="share"):
        calls[name]()
    assert not {"sixi_kv_read", "sixi_kv_attend", "sixi_kv_rope_apply"} & set(lib.calls)
    cache.append(one, one, b, stream=MAIN)  # (as inputs they are rows like others)
    rope.apply(one, Tensor((3,), I32), stream=MAIN)
    cache.attend(Expanded((3, 4, 32), BF), b, out=q, stream=MAIN)
