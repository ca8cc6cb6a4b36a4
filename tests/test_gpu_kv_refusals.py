"""What the cache's C entry points refuse before they launch anything: arrays that are not aligned to their elements."""

from __future__ import annotations

import ctypes

import pytest

from conftest import has_gpu

pytestmark = pytest.mark.gpu

if not has_gpu():
    pytest.skip("no CUDA device", allow_module_level=True)

import torch  # noqa: E402

import sixi_smp as S  # noqa: E402
from sixi_smp import kv_cache as K  # noqa: E402

DEV = torch.device("cuda:0")


class Call:
    """A call's arguments, one address of which may be moved."""

    def __init__(self):
        self.kv = K.KvCache(4, 16, 2, 32, device=0, max_seqs=4)
        self.rope = K.Rope(32, device=0)
        self.x = torch.zeros((3, 2, 32), device=DEV)
        self.table = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4)
        self.offsets, self.lens = torch.tensor([0, 3], device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
        self.positions = torch.arange(3, dtype=torch.int32, device=DEV)
        self.status, self.lse = torch.empty(1, dtype=torch.int32, device=DEV), torch.empty((3, 2), device=DEV)

    def __call__(self, name, moved=None, by=0):
        def at(what):
            return getattr(self, what).data_ptr() + (by if what == moved else 0)

        lib = S.load()
        t = K.KvTensor(at("x"), S.F32, 2, 64, 32)
        b = K.KvBatchStruct(at("table"), 4, at("offsets"), at("lens"), 1, 4, 3, 3)
        x, b = ctypes.byref(t), ctypes.byref(b)
        if name == "append":
            return lib.sixi_kv_append(self.kv.h, x, x, b, None, at("status"), None)
        if name == "read":
            return lib.sixi_kv_read(self.kv.h, b, x, x, at("status"), None)
        if name == "attend":
            return lib.sixi_kv_attend(self.kv.h, x, b, 1.0, 0, 0, None, x, at("lse"), at("status"), None)
        return lib.sixi_kv_rope_apply(self.rope.h, x, at("positions"), 3, 32, 0, x, None)


@pytest.mark.parametrize("name,arrays", [
    ("append", ["x", "table", "offsets", "lens", "status"]), ("read", ["x", "table", "offsets", "lens", "status"]),
    ("attend", ["x", "table", "offsets", "lens", "status", "lse"]), ("rope", ["x", "positions"])])
def test_misaligned_arrays_are_refused(name, arrays):
    call = Call()
    assert call(name) == 0
    for what in arrays:
        for by in (1, 2, 4) if what == "offsets" else (1, 2):
            assert call(name, what, by) == S.INVALID_ARGUMENT, (what, by)
    assert call(name) == 0
    torch.cuda.synchronize()
