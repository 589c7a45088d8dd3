"""What chunk_attn, the pool's operators and verify refuse before any launch: through the C ABI, with buffers that are never
touched, and by their Python arguments."""

import pytest
import torch

from qwenny_amd import Gemm, KvPool, TreeStep, kv_plan, kv_release
from qwenny_amd._lib import KvC, KvPoolC, TreeC, lib

FAKE = 0x10000  # a 16-byte aligned address that nothing reads


def _refused(rc, text):
    assert rc == -1, rc
    assert text in lib().qh_last_error().decode(), lib().qh_last_error().decode()


def _kv(**kw):
    return KvC(**{**dict(fmt=1, heads=4, head_dim=128, page=64, pages=8, codes=FAKE, scales=FAKE), **kw})


def _step(**kw):
    return TreeC(**{**dict(n=100, n_seq=1, max_new=100, start=FAKE, len=FAKE, table=FAKE, table_ld=4, mask=None), **kw})


def _chunk(step=None, q=FAKE, heads=8, scale=0.1, gate=None, out=FAKE, kv=None):
    return lib().qh_chunk_attn(None, None, q, heads, kv or _kv(), step or _step(), scale, gate, out)


def test_chunk_attn_refuses():
    assert _chunk(_step(n=0)) == 0 and _chunk(_step(n_seq=0)) == 0
    for heads in (6, 0, -4, 4 * 65):
        _refused(_chunk(heads=heads), "query heads")
    for name in ("start", "len", "table"):
        _refused(_chunk(_step(**{name: None})), "null")
    _refused(_chunk(q=None), "null")
    _refused(_chunk(out=None), "null")
    _refused(_chunk(_step(mask=FAKE)), "mask")
    _refused(_chunk(q=FAKE + 2), "aligned")
    _refused(_chunk(out=FAKE + 8), "aligned")
    _refused(_chunk(gate=FAKE + 4), "aligned")
    _refused(_chunk(_step(n_seq=-1)), "sequences")
    _refused(_chunk(_step(n_seq=1025)), "sequences")
    _refused(_chunk(_step(max_new=0)), "tokens")
    _refused(_chunk(_step(n=101)), "tokens")
    _refused(_chunk(_step(n=(1 << 20) + 1, max_new=1 << 21)), "2^20")
    _refused(_chunk(_step(table_ld=0)), "positions")
    _refused(_chunk(_step(table_ld=(1 << 24) + 1)), "positions")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _refused(_chunk(scale=scale), "scale")
    for change, text in (({"fmt": 3}, "format"), ({"head_dim": 96}, "dimensions"), ({"page": 96}, "pages of"), ({"codes": FAKE + 8}, "aligned"),
                         ({"scales": None}, "null cache"), ({"heads": 0}, "kv heads"), ({"pages": 1 << 26}, "31-bit")):
        _refused(_chunk(kv=_kv(**change)), text)
    assert lib().qh_chunk_attn(None, None, FAKE, 8, _kv(), None, 1.0, None, FAKE) == -1
    _refused(_chunk(), "null context")


def _pool(**kw):
    return KvPoolC(**{**dict(page=64, n_seq=3, pages=8, free=FAKE, n_free=FAKE, table=FAKE, table_ld=4, held=FAKE), **kw})


@pytest.mark.parametrize("change,text", [({"page": 32}, "pages of"), ({"page": 96}, "pages of"), ({"page": 2048}, "pages of"),
                                         ({"n_seq": 0}, "sequences"), ({"n_seq": 1025}, "sequences"), ({"pages": 0}, "31-bit"),
                                         ({"pages": 1 << 26}, "31-bit"), ({"table_ld": 0}, "positions"), ({"table_ld": (1 << 24) + 1}, "positions"),
                                         ({"free": None}, "null"), ({"n_free": None}, "null"), ({"table": None}, "null"), ({"held": None}, "null")])
def test_pools_refused(change, text):
    _refused(lib().qh_kv_release(None, _pool(**change), FAKE), text)
    _refused(lib().qh_kv_plan(None, _pool(**change), FAKE, FAKE, None, 1, FAKE, FAKE, FAKE, FAKE), text)


def test_plan_refuses():
    assert lib().qh_kv_release(None, None, FAKE) == -1
    _refused(lib().qh_kv_release(None, _pool(), None), "null")
    for k in range(6):
        args = [FAKE, FAKE, None, 1, FAKE, FAKE, FAKE, FAKE]
        args[(0, 1, 4, 5, 6, 7)[k]] = None
        _refused(lib().qh_kv_plan(None, _pool(), *args), "null")
    _refused(lib().qh_kv_plan(None, _pool(), FAKE, FAKE, None, (1 << 30) + 1, FAKE, FAKE, FAKE, FAKE), "2^30")


def _verify(step=None, logits=FAKE, ld=1000, vocab=1000, page=64, tokens=FAKE, draft=None, draft_ld=0, temp=None, u=FAKE, nxt=FAKE, count=FAKE,
            emit=FAKE, src=None, dst=None, new_len=None):
    return lib().qh_verify(None, None, logits, ld, vocab, step or _step(n=5, max_new=5), page, tokens, draft, draft_ld, temp, u, nxt, count,
                           emit, src, dst, new_len)


def test_verify_refuses():
    assert _verify(_step(n=0)) == 0 and _verify(_step(n_seq=0)) == 0
    for name in ("logits", "tokens", "u", "nxt", "count", "emit"):
        _refused(_verify(**{name: None}), "null")
    for name in ("start", "len"):
        _refused(_verify(_step(n=5, max_new=5, **{name: None})), "null")
    _refused(_verify(src=FAKE), "both")
    _refused(_verify(dst=FAKE), "both")
    _refused(_verify(_step(n=5, max_new=5, table=None), src=FAKE, dst=FAKE), "tables")
    for vocab in (0, (1 << 22) + 1):
        _refused(_verify(vocab=vocab, ld=1 << 23), "logits")
    _refused(_verify(ld=999), "vocabulary")
    _refused(_verify(draft=FAKE, draft_ld=999), "vocabulary")
    _refused(_verify(_step(n=5, max_new=65)), "tokens")
    _refused(_verify(_step(n=6, max_new=5)), "tokens")
    _refused(_verify(_step(n=5, max_new=0)), "tokens")
    _refused(_verify(_step(n=5, max_new=5, n_seq=1025)), "sequences")
    _refused(_verify(_step(n=5, max_new=5, n_seq=-2)), "sequences")
    for page in (0, 63, 96, 2048):
        _refused(_verify(page=page), "pages of")
    _refused(_verify(_step(n=5, max_new=5, table_ld=0)), "positions")
    _refused(_verify(_step(n=5, max_new=5, mask=FAKE), draft=FAKE, draft_ld=1000), "chains")
    _refused(_verify(), "null context")


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_python_types_refused():
    """torch makes int64 of whole numbers: read as int32 they would be pairs."""
    pool = KvPool.new(64, 10, 3, 4, device="cpu")
    assert pool.free.tolist() == list(range(9, -1, -1)) and pool.n_free.item() == 10
    for bad in (dict(free=_i32(10).long()), dict(table=_i32(4, 3).T), dict(held=_i32(2)), dict(n_free=_i32(1).float())):
        with pytest.raises(ValueError):
            KvPool(64, **{**dict(free=_i32(10), n_free=_i32(1), table=_i32(3, 4), held=_i32(3)), **bad})
    with pytest.raises(ValueError, match="len"):
        kv_release(0, pool, _i32(3).long())
    good = dict(len=_i32(3), add=_i32(3), start=_i32(4), slots=_i32(7), pos=_i32(7), granted=_i32(3))
    for name, t in good.items():
        for bad in (t.long(), t[:-1], t.repeat(2)[::2]):
            with pytest.raises(ValueError, match=name):
                kv_plan(0, pool, n=7, **{**good, name: bad})
    for bad in (torch.zeros(7), torch.zeros(6, dtype=torch.int64), torch.zeros(14, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="mask"):
            kv_plan(0, pool, n=7, mask=bad, **good)


def test_verify_arrays_refused():
    step = TreeStep(5, _i32(2), _i32(1), _i32(1, 4), 5)
    good = dict(logits=torch.zeros(5, 20), tokens=_i32(5), u=torch.zeros(5, 2), next=_i32(1), count=_i32(1), emit=_i32(5), temp=torch.zeros(1),
                draft=torch.zeros(5, 20), src=_i32(5), dst=_i32(5), new_len=_i32(1))
    bad = dict(logits=[torch.zeros(5, 19), torch.zeros(4, 20), torch.zeros(20, 5).T, torch.zeros(5, 20).half(), torch.zeros(100)],
               draft=[torch.zeros(5, 19), torch.zeros(5, 20).double()], tokens=[_i32(4), _i32(5).long(), None], u=[torch.zeros(9), torch.zeros(10).double()],
               temp=[torch.zeros(0), torch.zeros(1).double()], next=[_i32(0), None], count=[_i32(1).long()], emit=[_i32(10)[::2]], src=[_i32(4)],
               dst=[_i32(5).float()], new_len=[_i32(0)])
    gemm = Gemm.__new__(Gemm)  # (no context: nothing is launched)
    gemm._ctx = None
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError, match=name):
                gemm.verify(0, vocab=20, step=step, page=64, **{**good, name: value})
