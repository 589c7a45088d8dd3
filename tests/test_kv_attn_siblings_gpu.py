"""A token that a row does not see takes nothing from the row's output, however large its value: the row's probabilities are
rounded relative to the values that it sees."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvFmt, kv_write
from tests.test_kv_attn_forms_gpu import Wide
from tests.test_kv_attn_gpu import Step

pytestmark = pytest.mark.gpu


# d, query heads to a kv head, cached, tokens: chunks of 16 and 32 rows, four and eight waves, the step's tokens within one tile and
# over tiles' and turns' borders, results written directly and joined
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("form", [Step, Wide])
@pytest.mark.parametrize("d,h,old,tokens", [(128, 4, 100, 4), (64, 3, 0, 5), (256, 6, 250, 9), (256, 6, 900, 5), (128, 7, 2100, 31),
                                            (256, 7, 511, 64), (64, 16, 440, 40)])
@pytest.mark.parametrize("size", [2.0**24, 2.0**90])
def test_values_that_are_not_seen(gemm, fmt, form, d, h, old, tokens, size):
    print(f"{form.__name__} {fmt!r} {h}x{d} {old}+{tokens} {size}", flush=True)
    s = form([(old, tokens)], fmt, h, 1, d, 64, mask="tree")
    s.mask[:] = [1 << i for i in range(tokens)]  # each sees the cached positions and itself
    s.check(gemm)
    clean = s.run(gemm)
    large = [1, tokens - 1]
    s.v[[old + i for i in large]] *= size
    kv_write(None, s.kv, s.k, s.v, s.every, old + tokens)
    out = s.run(gemm)
    others = [i for i in range(tokens) if i not in large]
    assert torch.equal(out[others], clean[others])
    assert out.isfinite().all()
    want, tol = s.want()
    got = out.double().cpu().numpy()
    assert (np.abs(got - want) <= tol)[large].all()


@pytest.mark.parametrize("fmt", list(KvFmt))
def test_values_that_a_chain_does_not_see_yet(gemm, fmt):
    """Rows of a chain share chunks with the rows behind them, whose values grow from token to token."""
    for old, tokens in ((0, 20), (300, 20), (1000, 60)):
        print(f"{fmt!r} {old}+{tokens}", flush=True)
        s = Step([(old, tokens)], fmt, 6, 1, 256, 64)
        sizes = 4.0 ** torch.arange(tokens, device="cuda")
        s.v[old:] *= sizes[:, None, None].to(s.v.dtype)
        kv_write(None, s.kv, s.k, s.v, s.every, old + tokens)
        out = s.run(gemm)
        s.check(gemm)
        for t in (0, 1, tokens // 2, tokens - 2):  # the same row without what comes behind it
            part = Step.__new__(Step)
            part.__dict__.update(s.__dict__)
            part.seqs, part.n, part.start = [(old, t + 1)], t + 1, np.array([0, t + 1], np.int32)
            part.q = s.q[:t + 1].contiguous()
            part.slots = [s.slots[0][:old + t + 1]]  # (the values behind it are not counted in the tolerance either)
            want, tol = part.want()
            assert (np.abs(out[t].double().cpu().numpy() - want[t]) <= tol[t]).all(), t
