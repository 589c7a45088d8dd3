"""The cache's kernels, attn_prep and the attention run without scratch memory: their registers hold what they work on."""

import os

import pytest

from qwenny_amd.build import LIB
from tests.test_kernel_resources import _kernels


@pytest.mark.skipif(not os.path.exists(LIB), reason="nothing built")
@pytest.mark.parametrize("kernel", ["kv_write_kernel", "kv_write_batch_kernel", "kv_read_kernel", "kv_read_batch_kernel",
                                    "kv_move_kernel", "attn_prep_kernel", "tree_attn_kernel", "join_kernel"])
def test_no_scratch(kernel):
    found = {n: r for n, r in _kernels(LIB).items() if f"{len(kernel)}{kernel}I" in n}
    assert found
    assert not {n: r for n, r in found.items() if r}
