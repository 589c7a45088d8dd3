"""A tree's positions from masks of any kind: a token's is the cached ones and the number of tokens that it sees before itself, whether or
not it sees itself."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvPool, kv_plan

pytestmark = pytest.mark.gpu


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("news,lens", [([6], [0]), ([64], [700]), ([70, 5], [3, 9]), ([1, 0, 64, 3], [0, 5, 63, 64]), ([64] * 80, [100] * 80)], ids=str)
@pytest.mark.parametrize("itself", ["seen", "unseen", "some", "any"])
def test_positions(news, lens, itself):
    """(Eighty sequences of 64: the tokens have a launch of their own.)"""
    rng = np.random.default_rng(len(news))
    n, masks, want = sum(news), [], []
    for m, old in zip(news, lens):
        for i in range(m):
            mask = int(rng.integers(0, 2**63)) * 2 + int(rng.integers(0, 2))
            if itself != "any":  # those before it, and itself or not
                mask &= (1 << min(i, 63)) - 1
                if i < 64 and (itself == "seen" or (itself == "some" and rng.random() < 0.5)):
                    mask |= 1 << i
            masks.append(mask)
            want.append(old + (bin(mask & ((1 << i) - 1)).count("1") if i < 64 else i))
    seqs = len(news)
    pool = KvPool.new(64, seqs * 20, seqs, 20)
    start, slots, pos, granted = (_i32([77] * k) for k in (seqs + 1, n, n, seqs))
    kv_plan(None, pool, _i32(lens), _i32(news), n, start, slots, pos, granted, mask=torch.from_numpy(np.array(masks, np.uint64).view(np.int64)).cuda())
    assert granted.all()
    assert pos.tolist() == want
