"""The pool's calls write nothing outside of their arrays, whatever counts, pages and lengths these hold: each array lies in the middle of
a buffer whose other words keep their value."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvPool, kv_plan, kv_release

pytestmark = pytest.mark.gpu

AROUND, GUARD = 5000, 0x5A5A5A5A
HUGE = 2**31 - 1


class Arrays:
    def __init__(self):
        self.all = []

    def __call__(self, values):
        values = np.asarray(values, np.int64).astype(np.int32)
        whole = torch.full((values.size + 2 * AROUND,), GUARD, dtype=torch.int32, device="cuda")
        inner = whole[AROUND:AROUND + values.size].view(values.shape)
        inner.copy_(torch.from_numpy(values))
        self.all.append((whole, values.size))
        return inner

    def check(self):
        torch.cuda.synchronize()
        for k, (whole, size) in enumerate(self.all):
            assert (whole[:AROUND] == GUARD).all() and (whole[AROUND + size:] == GUARD).all(), k


@pytest.mark.parametrize("n", [0, 1, 300, 4096, 4097, 6000])
@pytest.mark.parametrize("n_seq,width,pages", [(1, 1, 1), (3, 4, 10), (64, 3, 100), (1000, 2, 500), (1024, 7, 7)])
def test_nothing_is_written_outside(n, n_seq, width, pages):
    rng = np.random.default_rng(n + n_seq)
    for turn in range(6):
        print(f"{n} tokens, {n_seq} sequences, {pages} pages, turn {turn}", flush=True)
        a = Arrays()
        odd = lambda k, *some: np.where(rng.random(k) < 0.7, rng.integers(0, 64 * width + 1, k), rng.choice(some, k))  # noqa: E731, B023
        free = np.where(rng.random(pages) < 0.7, rng.integers(0, pages, pages), rng.choice([-1, pages, HUGE, -HUGE - 1], pages))
        table = np.where(rng.random((n_seq, width)) < 0.7, rng.integers(0, pages, (n_seq, width)), rng.choice([-1, pages, HUGE], (n_seq, width)))
        held = np.where(rng.random(n_seq) < 0.7, rng.integers(0, width + 1, n_seq), rng.choice([-1, width + 1, HUGE, -HUGE - 1], n_seq))
        n_free = [pages, pages // 2, 0, -5, pages + 1, HUGE][turn]
        pool = KvPool(64, a(free), a([n_free]), a(table), a(held))
        lens, add = a(odd(n_seq, -1, HUGE, 64 * width + 1, -HUGE - 1)), a(odd(n_seq, -1, HUGE, 0, -HUGE - 1))
        start, slots, pos, granted = a(np.zeros(n_seq + 1)), a(np.zeros(n)), a(np.zeros(n)), a(np.zeros(n_seq))
        mask = torch.from_numpy(rng.integers(-2**63, 2**63, max(n, 1))).cuda() if turn % 2 else None
        for k in range(2):
            kv_plan(None, pool, lens, add, n, start, slots, pos, granted, mask=mask)
            a.check()
            kv_release(None, pool, lens if k == 0 else a(np.full(n_seq, (0, -1, HUGE)[turn % 3])))
            a.check()
        assert ((slots >= -1) & (slots < pages * 64)).all()
        assert ((start >= 0) & (start <= n)).all() and (start.diff() >= 0).all()
        assert 0 <= int(pool.n_free) <= pages and ((pool.held >= 0) & (pool.held <= width)).all()
