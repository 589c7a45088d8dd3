"""The bound that is stated for the prompts' attention over values of very different scales."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvCache, KvFmt, TreeStep
from tests.test_chunk_attn_gpu import _f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,code,most", [(KvFmt.I8, 255, 127), (KvFmt.E4M3, 0x7E, 448)])
@pytest.mark.parametrize("wide", [0, 90])
@pytest.mark.parametrize("first", [0, 64])
def test_values_of_a_very_small_scale(gemm, fmt, code, most, wide, first):
    """Among 65 tokens of equal probability one has the scale 0.501 and nothing but zeros, another 1.5 * 2^-31 and the largest code: half a
    step of f16's smallest numbers off, times the code. That is below 2^-24 (e4m3: 2^-22) of the largest scale times the probability, beside
    the output's own rounding, 2^-8 of it, and 3 * 2^-11 of what the value adds, 2^-20 for the sums. (`first` cached tokens: tiles that all rows
    see whole, or a border.)"""
    d, n = 64, 65 - first
    zero = 128 if fmt == KvFmt.I8 else 0
    codes = torch.full((2, 1, 2, 64 * d), zero, dtype=torch.uint8)
    scales = torch.ones((2, 1, 2, 64))
    scales[0, 0, 1] = 0.1
    scales[0, 0, 1, 0], scales[0, 0, 1, 1] = 0.501, 1.5 * 2.0**-31
    codes[0, 0, 1].view(d, 64)[:, 1] = code  # (token 1 is byte 1 of each dimension's 64)
    kv = KvCache(fmt, 1, d, 64, codes.cuda(), scales.cuda())
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1] + [-1] * wide], **i32)
    step = TreeStep(n, torch.tensor([0, n], **i32), torch.tensor([first], **i32), table, n)
    q, out = torch.zeros((n, 1, d), dtype=torch.bfloat16, device="cuda"), torch.empty((n, 1, d), dtype=torch.bfloat16, device="cuda")
    gemm.chunk_attn(None, q, 1, kv, step, out)
    seen = np.arange(first, 65)[:, None, None] + 1
    want = np.where(seen > 1, most * 1.5 * 2.0**-31 / seen, 0.0)
    tol = (2.0**-24 if fmt == KvFmt.I8 else 2.0**-22) * float(np.float32(0.501)) / seen
    got = _f64(out)
    assert (np.abs(got - want) <= tol + want * (2.0**-8 + 3 * 2.0**-11 + 2.0**-20)).all(), np.abs(got - want).max()
