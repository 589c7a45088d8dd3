"""The verification of trees whose masks say no more than each token's parent, or more than its ancestors: a token's parent is the last
that it sees before itself, and nothing else of the mask counts."""

import numpy as np
import pytest

from tests.test_verify_gpu import Case, _chances, _choose

pytestmark = pytest.mark.gpu

KINDS = {
    "parents": lambda rng, i, parent, masks: 1 << parent | 1 << i,  # (but not what is above them)
    "parents alone": lambda rng, i, parent, masks: 1 << parent,  # not itself either
    "some above": lambda rng, i, parent, masks: (masks[parent] & int(rng.integers(0, 2**63))) | 1 << parent | 1 << i,
    "others too": lambda rng, i, parent, masks: (int(rng.integers(0, 2**63)) & ((1 << parent) - 1)) | 1 << parent | 1 << i,
    "and later ones": lambda rng, i, parent, masks: masks[parent] | 1 << i | (int(rng.integers(0, 2**63)) << i + 1) & (1 << 64) - 1,
}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("news", [[5], [64], [64, 1, 0, 33, 17]], ids=str)
def test_only_parents_count(gemm, kind, news):
    longest = 0
    for seed in range(6):
        print(f"{kind} {news} {seed}", flush=True)
        c = Case(news, 300, tree=True, seed=seed, sharp=4.0)
        rng = np.random.default_rng(seed)
        for b, m in enumerate(c.news):
            masks, a = [1], c.start[b]
            for i in range(1, m):
                parent = c.parents[a + i]
                masks.append(KINDS[kind](rng, i, parent, masks))
                if rng.random() < 0.9:
                    c.tokens[a + i] = _choose(_chances(c.logits[a + parent], c.temp[b]), c.u[a + parent, 1])
                c.parents[a + i] = (masks[i] & ((1 << i) - 1)).bit_length() - 1
            if m:
                c.masks[a:a + m] = np.array(masks, np.uint64)
        longest = max(longest, c.check(gemm)["count"].max())
    assert longest >= 2


def test_roots_besides_the_first(gemm):
    """A token that sees none before itself has no parent, and is not reached."""
    c = Case([4], 50, tree=True, temps=(0.0,))
    c.parents, c.masks = [-1, -1, 1, 0], np.array([1, 2, 6, 9], np.uint64)
    first = int(c.logits[0].argmax())
    c.tokens[:] = [9, first, int(c.logits[1].argmax()), first]
    want = c.check(gemm)
    assert want["count"][0] == 1 and want["src"][1] == c.table[0, (c.len[0] + 3) // 64] * 64 + (c.len[0] + 3) % 64
