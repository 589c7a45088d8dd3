"""The prompts' attention at the ends of its numbers' range: queries, keys and softmax scales whose product is ordinary while they are
not."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvFmt, kv_write
from tests.test_chunk_attn_gpu import FORMS, _dev

pytestmark = pytest.mark.gpu


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("q,k,scale", [(-110, 110, 0.0625), (-126, 100, 2.0**22), (-90, 0, 2.0**87), (-125, 0, 3e38), (-60, 60, 0.0625), (60, 60, 2.0**-124),
                                       (100, -100, 0.0625), (-110, 10, 2.0**96), (120, -100, 2.0**-24), (0, 0, 1e-40)], ids=str)
def test_products_of_small_and_large(gemm, form, fmt, d, q, k, scale):
    """Scores of a few units (or none) by queries of 2^q, keys of 2^k and a scale."""
    print(f"{fmt!r} x{d}: 2^{q} 2^{k} {scale}", flush=True)
    s = form([(70, 66), (0, 5)], fmt, 4, 2, d, 64)
    s.q = _dev(s.rng.standard_normal((s.n, 4, d)) * 2.0**q, torch.bfloat16)
    for slots in s.slots:
        keys = _dev(s.rng.standard_normal((len(slots), 2, d)) * 2.0**k, torch.bfloat16)
        values = _dev(s.rng.standard_normal((len(slots), 2, d)), torch.bfloat16)
        kv_write(None, s.kv, keys, values, _dev(slots.astype(np.int32)), len(slots))
    s.check(gemm, scale=scale)
