"""What Gemm.chunk_attn refuses of its tensors, without a GPU: queries of another type would be read as pairs of bf16, and of arrays that
are too short or not in one piece the kernel would read and write what is not theirs."""

import pytest
import torch

from qwenny_amd import Gemm, KvCache, KvFmt, TreeStep
from qwenny_amd._lib import QhError

BF16, I32 = torch.bfloat16, torch.int32
N, H, J, D = 5, 4, 2, 64


def _call(q_heads=H, **change):
    """(No context: a call whose arrays are right is refused by the library, for that.)"""
    gemm = Gemm.__new__(Gemm)
    gemm._ctx = None
    kv = KvCache(KvFmt.I8, J, D, 64, torch.zeros((2, J, 2, 64 * D), dtype=torch.uint8), torch.zeros((2, J, 2, 64)))
    step = TreeStep(N, torch.tensor([0, N], dtype=I32), torch.zeros(1, dtype=I32), torch.zeros((1, 2), dtype=I32), N)
    arrays = {**dict(q=_rows(), gate=_rows(), out=_rows()), **change}
    gemm.chunk_attn(0, arrays["q"], q_heads, kv, step, arrays["out"], gate=arrays["gate"])


def _rows(n=N, h=H, d=D, dtype=BF16):
    return torch.zeros((n, h, d), dtype=dtype)


def test_arrays_that_are_right():
    wide = torch.zeros(N * H * D + 8, dtype=BF16)
    for change in ({}, {"gate": None}, {"q": _rows(N + 3)}, {"out": _rows().view(N, H * D)}, {"q": wide[8:]}, {"q": 0x10000, "out": 0x20000, "gate": None}):
        with pytest.raises(QhError, match="null context"):
            _call(**change)


@pytest.mark.parametrize("name", ["q", "gate", "out"])
def test_arrays_that_are_wrong(name):
    for bad in (_rows(dtype=torch.float32), _rows(dtype=torch.float16), _rows(N - 1), _rows(h=H - 1), _rows(d=D - 8), _rows(2 * N)[::2],
                _rows(H, N).transpose(0, 1), torch.zeros((N, H, D + 8), dtype=BF16)[..., :D], torch.zeros((N, H, 1), dtype=BF16).expand(N, H, D)):
        with pytest.raises(ValueError, match=name):
            _call(**{name: bad})


def test_more_heads_than_the_queries_have():
    with pytest.raises(ValueError, match="q"):
        _call(q_heads=2 * H)


@pytest.mark.parametrize("name", ["q", "out"])
def test_arrays_that_are_missing(name):
    with pytest.raises(QhError, match="null"):
        _call(**{name: None})
