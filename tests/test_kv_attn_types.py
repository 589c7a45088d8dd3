"""What the cache's and the attention's Python objects refuse of their tensors, without a GPU: other types than the kernels read
(torch makes int64 of whole numbers; as int32 they would be pairs) and arrays that do not lie in one piece."""

import pytest
import torch

from qwenny_amd import KvCache, KvFmt, TreeStep

I32 = torch.int32
SHAPE = (2, 64, 64)  # heads, dimensions, page


def _ints(*v, dtype=I32):
    return torch.tensor(v, dtype=dtype)


def _step(**change):
    d = dict(start=_ints(0, 2, 3), len=_ints(5, 0), table=torch.zeros((2, 4), dtype=I32), mask=_ints(1, 3, 1, dtype=torch.int64))
    d.update(change)
    return TreeStep(3, d["start"], d["len"], d["table"], 2, d["mask"])


def test_steps_that_are_right():
    _step()
    _step(mask=None)
    _step(mask=_ints(1, 3, 1, 7, dtype=torch.int64))  # longer is fine
    _step(mask=_ints(1, 3, 1, dtype=torch.int64).view(torch.uint64))
    TreeStep(3, _ints(0, 3), _ints(5), torch.zeros((4, 8), dtype=I32)[:1], 3)
    assert _step().c.n_seq == 2 and _step().c.table_ld == 4


@pytest.mark.parametrize("name", ["start", "len", "table"])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.float32])
def test_types_of_a_step(name, dtype):
    right = {"start": _ints(0, 2, 3), "len": _ints(5, 0), "table": torch.zeros((2, 4), dtype=I32)}
    with pytest.raises(ValueError, match=f"{name}.*int32"):
        _step(**{name: right[name].to(dtype)})


@pytest.mark.parametrize("dtype", [torch.int32, torch.uint8, torch.float64])
def test_types_of_a_mask(dtype):
    with pytest.raises(ValueError, match="mask.*64"):
        _step(mask=torch.ones(3, dtype=dtype))


def test_strides_of_a_step():
    for name, array in (("start", torch.zeros(6, dtype=I32)[::2]), ("len", torch.zeros(4, dtype=I32)[::2]),
                        ("mask", torch.zeros(6, dtype=torch.int64)[::2])):
        with pytest.raises(ValueError, match=f"{name}.*contiguous"):
            _step(**{name: array})
    for table in (torch.zeros((4, 2), dtype=I32).t(), torch.zeros((2, 8), dtype=I32)[:, :4]):
        with pytest.raises(ValueError, match="table"):
            _step(table=table)


def test_caches():
    heads, d, page = SHAPE
    codes, scales = torch.zeros((3, heads, 2, page * d), dtype=torch.uint8), torch.zeros((3, heads, 2, page))
    make = lambda c, s: KvCache(KvFmt.E4M3, heads, d, page, c, s, 3)  # noqa: E731
    make(codes, scales)
    make(codes.view(torch.float8_e4m3fn), scales)  # (the same bytes)
    make(codes[:3], scales[:3])
    for bad in (codes.to(torch.int32), codes.to(torch.bfloat16)):
        with pytest.raises(ValueError, match="codes"):
            make(bad, scales)
    for bad in (scales.double(), torch.zeros((6, heads, 2, page), dtype=torch.float16)):
        with pytest.raises(ValueError, match="scales"):
            make(codes, bad)
    layers = torch.zeros((3, 5) + tuple(codes.shape[1:]), dtype=torch.uint8)  # a layer's pages lie apart
    with pytest.raises(ValueError, match="codes.*contiguous"):
        make(layers[:, 1], scales)
    with pytest.raises(ValueError, match="scales.*contiguous"):
        make(codes, torch.zeros((3, 5, heads, 2, page))[:, 1])
    with pytest.raises(ValueError, match="bytes"):
        make(codes[:2], scales)
