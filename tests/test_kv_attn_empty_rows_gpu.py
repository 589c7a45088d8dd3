"""A token that sees nothing gets zeros whatever its query holds: nothing is multiplied with it."""

import pytest
import torch

from qwenny_amd import KvFmt
from tests.test_kv_attn_forms_gpu import Wide
from tests.test_kv_attn_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("form", [Step, Wide])
@pytest.mark.parametrize("d,h,tokens", [(64, 2, 3), (256, 6, 9), (128, 7, 40)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite(gemm, fmt, form, d, h, tokens, bad):
    print(f"{form.__name__} {fmt!r} {h}x{d} {tokens} {bad}", flush=True)
    s = form([(0, tokens), (70, 2)], fmt, h, 1, d, 64, mask="tree", gate=True)
    s.mask[:tokens] = 0
    s.mask[1] = 2  # this one sees itself
    clean = s.run(gemm)
    s.q[0, :, 3], s.q[2, 1, d - 1] = bad, bad
    out = s.run(gemm)
    assert torch.equal(out, clean)
    assert (out[[i for i in range(tokens) if i != 1]] == 0).all() and out[1].isfinite().all()
    s.q[1, 0, 0] = bad  # what it sees it is multiplied with
    out = s.run(gemm)
    assert out[1, 0].isnan().all() and torch.equal(out[1, 1:], clean[1, 1:]) and torch.equal(out[2:], clean[2:])
