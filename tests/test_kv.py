"""CPU checks of the key/value cache's C boundary (include/sixi_kv.h): exported symbols, record
layouts, argument refusals before any device call, and the tests' own 64-bit reference."""

from __future__ import annotations

import ctypes
import re
import subprocess
import textwrap

import numpy as np
import pytest

import kv_reference as R
from conftest import REPO

HEADER = REPO / "include" / "sixi_kv.h"
LIB = REPO / "sixi-asi_b200" / "lib" / "libsixi_smp.so"
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: the calls below return before that


def declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(sixi_kv_[a-z_]+)\s*\(", text)))


def test_exports_and_binding_match_the_header():
    import sixi_smp

    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB)], capture_output=True, text=True, check=True).stdout
    assert sorted(set(re.findall(r"\bT (sixi_kv_\w+)", out))) == declared()
    assert sorted(sixi_smp.KV_SIGNATURES) == declared()
    lib = sixi_smp.load()
    assert all(hasattr(lib, n) for n in declared())


def test_record_layouts(tmp_path):
    from sixi_smp import kv_cache as K

    pairs = [("sixi_kv_config", K.KvConfig), ("sixi_kv_tensor", K.KvTensor), ("sixi_kv_batch", K.KvBatchStruct),
             ("sixi_kv_rope_config", K.RopeConfig)]
    lines = []
    for c, py in pairs:
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text(textwrap.dedent(f"""
        #include <stddef.h>
        #include <stdio.h>
        #include "{HEADER}"
        int main(void) {{ {' '.join(lines)} return 0; }}
    """))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, py in pairs:
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f[0]).offset for f in py._fields_]
    assert got == want


@pytest.mark.parametrize("change", [
    dict(page_size=8), dict(page_size=48), dict(page_size=256), dict(page_size=0), dict(n_pages=0), dict(n_kv_heads=0),
    dict(n_kv_heads=1025), dict(head_dim=0), dict(head_dim=24), dict(head_dim=272), dict(max_seqs=0),
    dict(max_seqs=65536), dict(n_pages=2 ** 31 - 1, n_kv_heads=2)])
def test_create_refuses(change):
    import sixi_smp
    from sixi_smp import kv_cache as K

    f = dict(n_pages=8, page_size=64, n_kv_heads=2, head_dim=64, max_seqs=16)
    f.update(change)
    c = K.KvConfig(f["n_pages"], f["page_size"], f["n_kv_heads"], f["head_dim"], f["max_seqs"], 0)
    h = ctypes.c_void_p()
    assert sixi_smp.load().sixi_kv_create(0, ctypes.byref(c), FAKE, FAKE, FAKE, FAKE, ctypes.byref(h)) == \
        sixi_smp.INVALID_ARGUMENT
    assert not h.value


def test_create_refuses_missing_and_misaligned_buffers():
    import sixi_smp
    from sixi_smp import kv_cache as K

    lib = sixi_smp.load()
    c = K.KvConfig(8, 64, 2, 64, 16, 0)
    h = ctypes.c_void_p()
    for i in range(4):
        for bad in (None, ctypes.c_void_p(0x1002)):
            p = [FAKE] * 4
            p[i] = bad
            assert lib.sixi_kv_create(0, ctypes.byref(c), *p, ctypes.byref(h)) == sixi_smp.INVALID_ARGUMENT
    assert lib.sixi_kv_create(0, None, FAKE, FAKE, FAKE, FAKE, ctypes.byref(h)) == sixi_smp.INVALID_ARGUMENT
    assert lib.sixi_kv_create(0, ctypes.byref(c), FAKE, FAKE, FAKE, FAKE, None) == sixi_smp.INVALID_ARGUMENT
    assert lib.sixi_kv_create(-1, ctypes.byref(c), FAKE, FAKE, FAKE, FAKE, ctypes.byref(h)) == sixi_smp.INVALID_ARGUMENT
    assert lib.sixi_kv_destroy(None) == 0


@pytest.mark.parametrize("change", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(layout=2), dict(scaling=4), dict(base=1.0),
    dict(base=float("nan")), dict(base=float("inf")), dict(scaling=1, factor=0.5), dict(scaling=1, factor=float("nan")),
    dict(scaling=2, factor=2.0, rot_dim=2), dict(scaling=3, factor=2.0, original_max_position=0),
    dict(scaling=3, factor=2.0, beta_slow=0.0), dict(scaling=3, factor=2.0, beta_slow=64.0)])
def test_rope_create_refuses(change):
    import sixi_smp
    from sixi_smp import kv_cache as K

    f = dict(rot_dim=64, layout=0, scaling=0, original_max_position=4096, base=10000.0, factor=1.0, beta_fast=32.0,
             beta_slow=1.0)
    f.update(change)
    c = K.RopeConfig(*f.values())
    h = ctypes.c_void_p()
    assert sixi_smp.load().sixi_kv_rope_create(0, ctypes.byref(c), ctypes.byref(h)) == sixi_smp.INVALID_ARGUMENT
    assert not h.value


def test_calls_refuse_a_missing_handle():
    import sixi_smp

    lib, inv = sixi_smp.load(), sixi_smp.INVALID_ARGUMENT
    assert lib.sixi_kv_rope_apply(None, FAKE, FAKE, 1, 64, 0, FAKE, None) == inv
    assert lib.sixi_kv_append(None, FAKE, FAKE, FAKE, None, FAKE, None) == inv
    assert lib.sixi_kv_read(None, FAKE, FAKE, FAKE, FAKE, None) == inv
    assert lib.sixi_kv_attend(None, FAKE, FAKE, 1.0, 0, 0, None, FAKE, FAKE, FAKE, None) == inv
    assert lib.sixi_kv_rope_destroy(None) == 0


def test_reference_rounding_is_e4m3():
    """The reference's own e4m3: every value rounds to itself, midpoints to the even one, torch agrees."""
    import torch

    fin = np.array([b for b in range(256) if b & 0x7F != 0x7F], np.uint8)
    assert np.array_equal(R.round_e4m3(R.E4M3[fin]), fin)
    v = R.E4M3[:0x7F]
    mid = (v[:-1] + v[1:]) / 2
    assert np.all(R.round_e4m3(mid) % 2 == 0)
    x = np.random.default_rng(1).normal(size=20000) * 30
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.round_e4m3(x.astype(np.float64)), want)


def test_reference_scale_rule():
    for e in (-126, -3, 0, 7, 119):
        assert R.scale_exp(448.0 * 2.0 ** e) == e
        assert R.scale_exp(np.nextafter(448.0 * 2.0 ** e, np.inf)) == e + 1
    assert R.scale_exp(0.0) == -126 and R.scale_exp(1e-45) == -126
