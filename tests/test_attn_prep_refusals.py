"""What attn_prep refuses of its norms' weights, without a GPU: the header asks for 16-byte alignment, and the kernel reads whole
vectors of them."""

import pytest

from qwenny_amd._lib import AttnRowsC, KvC, lib

FAKE = 0x10000


@pytest.mark.parametrize("which", ["q_w", "k_w"])
@pytest.mark.parametrize("offset", [2, 4, 8, 12])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_weights_off_their_alignment(which, offset, d):
    w = {"q_w": FAKE, "k_w": FAKE}
    w[which] += offset
    kv = KvC(fmt=1, heads=2, head_dim=d, page=64, pages=4, codes=FAKE, scales=FAKE)
    for cache, slots, k in ((kv, FAKE, None), (None, None, FAKE)):
        rc = lib().qh_attn_prep(None, FAKE, 1, 1, AttnRowsC(4, 2, d, 16, 0), w["q_w"], w["k_w"], 1e-6, FAKE, FAKE, FAKE, None, cache, slots, k, k)
        assert rc == -1 and "aligned" in lib().qh_last_error().decode()
