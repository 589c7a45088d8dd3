"""chunk_attn and verify write nothing outside of their arrays, whatever starts and lengths hold; new lengths may go where the old ones
lie."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvFmt, TreeStep
from tests.test_chunk_attn_gpu import FORMS
from tests.test_verify_gpu import Case, _dev

pytestmark = pytest.mark.gpu

AROUND = 5000
HUGE = 2**31 - 1
# starts of three sequences of 70, 3 and 100 tokens (or 7, 3 and 10), as far as they are that
STARTS = ["right", "short", [0, HUGE, -1, HUGE], [-HUGE - 1, -1, 0, 1], [5, 4, 3, 2], [0, 0, 0, 0]]


class Guarded:
    """An array in the middle of a buffer whose other elements keep their value."""

    def __init__(self, shape, dtype, guard):
        self.size, self.guard = int(np.prod(shape)), guard
        self.whole = torch.full((self.size + 2 * AROUND + 8,), guard, dtype=dtype, device="cuda")
        self.at = AROUND + 8 - AROUND % 8  # (16-byte aligned for two bytes each)
        self.inner = self.whole[self.at:self.at + self.size].view(shape)

    def check(self):
        assert (self.whole[:self.at] == self.guard).all() and (self.whole[self.at + self.size:] == self.guard).all()


def _starts(start, news):
    right = np.cumsum([0] + news)
    return right if start == "right" else np.minimum(right, right[-1] - 2) if start == "short" else np.array(start, np.int64)


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("start", STARTS, ids=str)
def test_chunk_attn_writes_nothing_outside(gemm, form, fmt, d, start):
    print(f"{fmt!r} x{d} {start}", flush=True)
    s = form([(100, 70), (300, 3), (4000, 100)], fmt, 6, 2, d, 64, gate=True)
    s.start = _starts(start, [70, 3, 100]).astype(np.int32)
    for lens in (s.len, [HUGE, -1, -HUGE - 1]):
        s.len = np.array(lens, np.int64).astype(np.int32)
        out = Guarded((s.n, s.h, s.d), torch.bfloat16, 55.0)
        gemm.chunk_attn(None, s.q, s.h, s.kv, s.step(), out.inner, gate=s.gate)
        out.check()
        assert not (out.inner == 55.0).all(-1).any()  # every row is written


@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
@pytest.mark.parametrize("start", STARTS, ids=str)
def test_verify_writes_nothing_outside(gemm, kind, start):
    print(f"{kind} {start}", flush=True)
    c = Case([7, 3, 10], 5000, tree=kind == "tree", draft=kind == "draft")
    c.start = _starts(start, [7, 3, 10]).astype(np.int32)
    for lens in (c.len, [HUGE, -1, 3]):
        c.len = np.array(lens, np.int64).astype(np.int32)
        out = {k: Guarded((n,), torch.int32, 77) for k, n in (("next", 3), ("count", 3), ("emit", 20), ("src", 20), ("dst", 20), ("new_len", 3))}
        c.run(gemm, out={k: g.inner for k, g in out.items()})
        for g in out.values():
            g.check()
        assert ((out["emit"].inner >= -1) & (out["emit"].inner < 5000)).all()


@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
def test_new_lengths_in_place(gemm, kind):
    """A program that keeps one array of lengths has the new ones written over the old."""
    c = Case([5, 0, 3, 8, 1], 3000, tree=kind == "tree", draft=kind == "draft", temps=(0.8, 1.0, 1.3))
    want, lens = c.want(), _dev(c.len)
    step = TreeStep(c.n, _dev(c.start), lens, _dev(c.table), 8, None if c.masks is None else _dev(c.masks.view(np.int64)))
    out = c.buffers()
    out["new_len"] = lens
    got = c.run(gemm, step=step, out=out)
    for name, w in want.items():
        assert np.array_equal(got[name].cpu().numpy(), w), name
