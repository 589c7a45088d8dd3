"""Arrays that are missing, or that are addresses without a type, refused by name in the pool's calls and in verify, without a GPU."""

import pytest
import torch

from qwenny_amd import Gemm, KvPool, TreeStep, kv_plan, kv_release


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("value", [None, 0x10000, [0, 0, 0]], ids=str)
def test_a_pools_calls(value):
    pool = KvPool.new(64, 10, 3, 4, device="cpu")
    for name in ("free", "n_free", "held"):
        with pytest.raises(ValueError, match=name):
            KvPool(64, **{**dict(free=_i32(10), n_free=_i32(1), table=_i32(3, 4), held=_i32(3)), name: value})
    with pytest.raises(ValueError, match="len"):
        kv_release(0, pool, value)
    good = dict(len=_i32(3), add=_i32(3), start=_i32(4), slots=_i32(7), pos=_i32(7), granted=_i32(3))
    for name in good:
        with pytest.raises(ValueError, match=name):
            kv_plan(0, pool, n=7, **{**good, name: value})
    if value is not None:
        with pytest.raises(ValueError, match="mask"):
            kv_plan(0, pool, n=7, mask=value, **good)


@pytest.mark.parametrize("value", [None, 0x10000, [0.0]], ids=str)
def test_verify(value):
    step = TreeStep(5, _i32(2), _i32(1), _i32(1, 4), 5)
    good = dict(logits=torch.zeros(5, 20), tokens=_i32(5), u=torch.zeros(5, 2), next=_i32(1), count=_i32(1), emit=_i32(5))
    more = dict(temp=torch.zeros(1), draft=torch.zeros(5, 20), src=_i32(5), dst=_i32(5), new_len=_i32(1))
    gemm = Gemm.__new__(Gemm)
    gemm._ctx = None
    for name in (*good, *(more if value is not None else ())):
        with pytest.raises(ValueError, match=name):
            gemm.verify(0, vocab=20, step=step, page=64, **{**good, **more, name: value})
