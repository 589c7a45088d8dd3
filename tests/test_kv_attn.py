"""The decode step's attention without a GPU: the work plan of the kernels walked on the CPU under sanitizers, and what the
entry points refuse before any launch (through the C ABI, with buffers that are never touched)."""

import ctypes
import os
import shutil
import subprocess

import pytest

from qwenny_amd import KvCache, KvFmt
from qwenny_amd._lib import AttnRowsC, KvC, QhError, TreeC, lib

HERE = os.path.dirname(os.path.abspath(__file__))
FAKE = 0x10000  # a 16-byte aligned address that nothing reads


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_work_plan_under_sanitizers(tmp_path):
    exe = str(tmp_path / "driver")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(HERE, "attn_plan_driver.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def _kv(**kw):
    d = dict(fmt=1, heads=4, head_dim=128, page=64, pages=8, codes=FAKE, scales=FAKE)
    d.update(kw)
    return KvC(**d)


def _refused(rc, text):
    assert rc == -1, rc
    assert text in lib().qh_last_error().decode(), lib().qh_last_error().decode()


BAD_CACHES = [({"fmt": 0}, "format"), ({"fmt": 3}, "format"), ({"head_dim": 96}, "dimensions"), ({"head_dim": 0}, "dimensions"),
              ({"page": 32}, "pages of"), ({"page": 96}, "pages of"), ({"page": 2048}, "pages of"), ({"page": -64}, "pages of"),
              ({"heads": 0}, "kv heads"), ({"heads": -1}, "kv heads"), ({"pages": 0}, "31-bit"), ({"pages": 1 << 26}, "31-bit")]


@pytest.mark.parametrize("change,text", BAD_CACHES)
def test_cache_descriptions_refused(change, text):
    kv = _kv(**change)
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    _refused(lib().qh_kv_sizes(kv, ctypes.byref(a), ctypes.byref(b)), text)
    _refused(lib().qh_kv_write(None, kv, FAKE, FAKE, FAKE, 1), text)
    _refused(lib().qh_kv_read(None, kv, FAKE, 1, FAKE, FAKE), text)
    _refused(lib().qh_kv_move(None, kv, FAKE, FAKE, 1, FAKE, 1), text)
    _refused(lib().qh_tree_attn(None, None, FAKE, 8, kv, _tree(), 1.0, None, FAKE), text)


def test_cache_buffers_refused():
    for change in ({"codes": None}, {"scales": None}):
        _refused(lib().qh_kv_write(None, _kv(**change), FAKE, FAKE, FAKE, 1), "null cache")
    for change in ({"codes": FAKE + 8}, {"scales": FAKE + 4}):
        _refused(lib().qh_kv_read(None, _kv(**change), FAKE, 1, FAKE, FAKE), "aligned")


def test_cache_operators_refuse():
    kv = _kv()
    assert lib().qh_kv_write(None, kv, None, None, None, 0) == 0  # nothing to do
    assert lib().qh_kv_read(None, kv, None, 0, None, None) == 0
    assert lib().qh_kv_move(None, kv, None, None, 0, None, 3) == 0
    _refused(lib().qh_kv_write(None, kv, None, FAKE, FAKE, 1), "null")
    _refused(lib().qh_kv_write(None, kv, FAKE, FAKE, None, 1), "null")
    _refused(lib().qh_kv_write(None, kv, FAKE + 2, FAKE, FAKE, 1), "aligned")
    _refused(lib().qh_kv_write(None, kv, FAKE, FAKE, FAKE, (1 << 20) + 1), "tokens")
    _refused(lib().qh_kv_read(None, kv, None, 1, FAKE, FAKE), "null")
    _refused(lib().qh_kv_read(None, kv, FAKE, 1, FAKE, FAKE + 8), "aligned")
    _refused(lib().qh_kv_move(None, kv, FAKE, None, 1, FAKE, 1), "null")
    _refused(lib().qh_kv_move(None, kv, FAKE, FAKE, 1, FAKE, -1), "sequences")


def _prep(rows=None, splits=1, n=1, x=FAKE, kv=None, slots=None, k=FAKE, v=FAKE, q=FAKE, gate=None, inv=FAKE, pos=FAKE):
    r = dict(q_heads=8, kv_heads=4, head_dim=128, rot=64, gated=0)
    r.update(rows or {})
    return lib().qh_attn_prep(None, x, splits, n, AttnRowsC(**r), FAKE, FAKE, 1e-6, inv, pos, q, gate, kv, slots, k, v)


def test_attn_prep_refuses():
    assert _prep(n=0) == 0
    _refused(_prep({"head_dim": 80}), "dimensions")
    _refused(_prep({"rot": 130}), "rotated")
    _refused(_prep({"rot": 63}), "rotated")
    _refused(_prep({"rot": -2}), "rotated")
    _refused(_prep({"kv_heads": 0}), "heads")
    _refused(_prep(splits=0), "splits")
    _refused(_prep(x=None), "null")
    _refused(_prep(x=FAKE + 4), "aligned")
    _refused(_prep(k=None), "null")
    _refused(_prep({"gated": 1}), "null")
    _refused(_prep(inv=None), "null")
    _refused(_prep(pos=None), "null")
    _refused(_prep(kv=_kv(), slots=None), "null")
    _refused(_prep(kv=_kv(heads=2), slots=FAKE), "a cache of")
    _refused(_prep(kv=_kv(head_dim=64), slots=FAKE), "a cache of")
    _refused(_prep(kv=_kv(page=65), slots=FAKE), "pages of")


def _tree(**kw):
    d = dict(n=1, n_seq=1, max_new=1, start=FAKE, len=FAKE, table=FAKE, table_ld=4, mask=None)
    d.update(kw)
    return TreeC(**d)


def _attn(step=None, q=FAKE, heads=8, scale=0.1, gate=None, out=FAKE, kv=None):
    return lib().qh_tree_attn(None, None, q, heads, kv or _kv(), step or _tree(), scale, gate, out)


def test_tree_attn_refuses():
    assert _attn(_tree(n=0)) == 0 and _attn(_tree(n_seq=0)) == 0
    _refused(_attn(heads=6), "query heads")
    _refused(_attn(heads=0), "query heads")
    _refused(_attn(heads=4 * 65), "query heads")
    for name in ("start", "len", "table"):
        _refused(_attn(_tree(**{name: None})), "null")
    _refused(_attn(q=None), "null")
    _refused(_attn(out=None), "null")
    _refused(_attn(out=FAKE + 2), "aligned")
    _refused(_attn(gate=FAKE + 8), "aligned")
    _refused(_attn(_tree(n_seq=-1)), "sequences")
    _refused(_attn(_tree(n_seq=1025)), "sequences")
    _refused(_attn(_tree(max_new=0)), "tokens")
    _refused(_attn(_tree(max_new=65)), "tokens")
    _refused(_attn(_tree(n=3, n_seq=2)), "tokens")
    _refused(_attn(_tree(table_ld=0)), "positions")
    _refused(_attn(_tree(table_ld=(1 << 24) + 1)), "positions")
    _refused(_attn(_tree(table_ld=1 << 24, n_seq=1024)), "too many")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _refused(_attn(scale=scale), "scale")
    _refused(_attn(), "null context")


def test_cache_sizes():
    assert KvCache.sizes(KvFmt.I8, 4, 256, 256, 10) == (10 * 4 * 2 * 256 * 256, 10 * 4 * 2 * 256 * 4)
    with pytest.raises(QhError):
        KvCache.sizes(KvFmt.E4M3, 4, 256, 100, 10)
