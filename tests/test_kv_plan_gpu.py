"""The pool of pages on the GPU against a list that requests push to and pop from: whole numbers, all of them equal."""

import numpy as np
import pytest
import torch

from qwenny_amd import Graph, KvPool, kv_plan, kv_release

pytestmark = pytest.mark.gpu


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


class Pool:
    """A pool on the GPU, and its double on the host."""

    def __init__(self, page, pages, n_seq, width, seed=0):
        self.page, self.pages, self.n_seq, self.width = page, pages, n_seq, width
        rng = np.random.default_rng(seed)
        self.free, self.n_free = rng.permutation(pages).astype(np.int64), pages
        self.table, self.held = np.full((n_seq, width), -1, np.int64), np.zeros(n_seq, np.int64)
        self.dev = KvPool(page, _dev(self.free), _dev([pages]), _dev(self.table), _dev(self.held))

    def release(self, lens):
        kv_release(None, self.dev, _dev(lens))
        for b in reversed(range(self.n_seq)):
            keep = -(-int(lens[b]) // self.page) if lens[b] >= 0 else self.held[b]
            while self.held[b] > keep:
                self.held[b] -= 1
                self.free[self.n_free] = self.table[b, self.held[b]]
                self.table[b, self.held[b]] = -1
                self.n_free += 1

    def plan(self, lens, add, n, mask=None):
        start, slots, pos, granted = (torch.full((k,), 77, dtype=torch.int32, device="cuda") for k in (self.n_seq + 1, n, n, self.n_seq))
        kv_plan(None, self.dev, _dev(lens), _dev(add), n, start, slots, pos, granted,
                mask=None if mask is None else torch.from_numpy(mask.view(np.int64)).cuda())
        want = [np.zeros(self.n_seq + 1, np.int64), np.full(n, -1, np.int64), np.zeros(n, np.int64), np.zeros(self.n_seq, np.int64)]
        asked, there, at = 0, self.n_free, 0
        for b, (a, m) in enumerate(zip(map(int, lens), map(int, add))):
            fits = a >= 0 and m >= 0 and a + m <= self.width * self.page
            need = max(0, -(-(a + m) // self.page) - self.held[b]) if fits and m > 0 else 0
            asked += need
            ok = fits and (need == 0 or asked <= there)
            for _ in range(need if ok else 0):
                self.n_free -= 1
                self.table[b, self.held[b]] = self.free[self.n_free]
                self.held[b] += 1
            for i in range(max(min(m, n - at), 0)):
                if ok:
                    want[1][at + i] = self.table[b, (a + i) // self.page] * self.page + (a + i) % self.page
                depth = i if mask is None or i >= 64 else max(bin(int(mask[at + i]) & ((2 << i) - 1)).count("1") - 1, 0)
                want[2][at + i] = min(a + depth, 2**31 - 1)  # (as far as an int32 goes)
            at += max(m, 0)
            want[0][b + 1] = min(at, n)
            want[3][b] = ok
        return [start, slots, pos, granted], want

    def check(self):
        assert int(self.dev.n_free) == self.n_free
        for name in ("free", "table", "held"):
            assert np.array_equal(getattr(self.dev, name).cpu().numpy(), getattr(self, name)), name


def _equal(got, want):
    for name, g, w in zip(("start", "slots", "pos", "granted"), got, want):
        g = g.cpu().numpy()
        assert np.array_equal(g, w), (name, np.flatnonzero(g != w)[:5], g[g != w][:5], w[g != w][:5])


@pytest.mark.parametrize("n_seq,page,most,tokens", [(1, 64, 500, 1), (1, 256, 5000, 5), (3, 64, 300, 200), (16, 256, 9000, 2000), (64, 64, 900, 8),
                                                    (65, 128, 900, 8), (1000, 64, 2000, 5), (1024, 1024, 9000, 1)])
def test_a_server_run(n_seq, page, most, tokens):
    """Requests come, grow, lose rejected drafts and end; sometimes there are not pages enough."""
    rng = np.random.default_rng(n_seq)
    width = -(-(most + tokens) // page) + 1
    pool = Pool(page, max(2, int(n_seq * width * 0.5)), n_seq, width, seed=n_seq)
    lens = np.zeros(n_seq, np.int64)
    denied = 0
    for turn in range(8):
        print(f"{n_seq} sequences, turn {turn}", flush=True)
        add = np.where(rng.random(n_seq) < 0.8, rng.integers(1, tokens + 1, n_seq), 0)
        fresh = (lens == 0) & (rng.random(n_seq) < 0.7)
        add[fresh] = rng.integers(1, tokens + 1, fresh.sum())
        n = int(add.sum()) + (turn % 3) * 5
        if n == 0:
            n = 1
        got, want = pool.plan(lens, add, n)
        _equal(got, want)
        pool.check()
        ok = want[3] == 1
        denied += int((~ok).sum())
        kept = np.where(ok & (add > 0), lens + rng.integers(0, add + 1), lens)
        kept[rng.random(n_seq) < 0.15] = 0
        lens = np.minimum(kept, most)
        pool.release(lens)
        pool.check()
    assert sorted(list(pool.free[:pool.n_free]) + list(pool.table[pool.table >= 0])) == list(range(pool.pages))


def test_not_enough_pages():
    """From the first sequence that cannot be served on, those that need pages get none; those that need none go on."""
    pool = Pool(64, 5, 6, 8)
    got, want = pool.plan([0, 0, 0, 0, 0, 0], [64, 100, 200, 10, 0, 10], 384)
    assert want[3].tolist() == [1, 1, 0, 0, 1, 0]
    _equal(got, want)
    pool.check()
    got, want = pool.plan([64, 100, 0, 0, 0, 0], [1, 28, 0, 300, 0, 64], 400)
    assert want[3].tolist() == [1, 1, 1, 0, 1, 0]
    _equal(got, want)
    pool.check()


def test_numbers_that_do_not_fit():
    pool = Pool(64, 50, 6, 4)
    big = 2**31 - 1
    got, want = pool.plan([-1, 256, 250, big, 5, 0], [3, 1, 6, big, -7, 9], 19)
    assert want[3].tolist() == [0, 0, 1, 0, 0, 1]
    _equal(got, want)
    pool.check()
    pool.release([-1, -5, 0, -1, 0, big])
    pool.check()


def test_a_release_undoes_a_plan():
    pool = Pool(64, 100, 7, 20)
    lens = np.array([0, 64, 65, 1, 0, 300, 7])
    pool.plan(np.zeros(7, np.int64), lens, int(lens.sum()))
    before = pool.dev.free.clone()
    for _ in range(2):
        pool.plan(lens, [70, 1, 0, 200, 3, 30, 64], 368)
        pool.release(lens)
        pool.check()
        assert torch.equal(before, pool.dev.free)


@pytest.mark.parametrize("n_seq,tokens", [(1, 64), (5, 13), (200, 8), (300, 64)])
def test_trees(n_seq, tokens):
    """A tree's tokens lie one after the other, their positions are their depths; a token that sees nothing counts as a root."""
    rng = np.random.default_rng(tokens)
    add = rng.integers(0, tokens + 1, n_seq)
    add[0] = tokens
    mask = []
    for m in add:
        for i in range(m):
            parent = int(rng.integers(-1, i)) if i else -1
            mask.append((mask[len(mask) - i + parent] if parent >= 0 else 0) | 1 << i)
    mask = np.array(mask, np.uint64)
    if len(mask) > 5:
        mask[5] = 0
    pool = Pool(64, n_seq * 20, n_seq, 20)
    got, want = pool.plan(rng.integers(0, 900, n_seq), add, len(mask), mask)
    _equal(got, want)


@pytest.mark.parametrize("n", [4095, 4096, 4097, 40000])
def test_token_counts(n):
    """Steps of one launch and of two; tokens that the sequences have not, and sequences that the step has not room for."""
    for total in (n, n - 100, n + 100):
        add = np.array([total // 3, 0, 17, total - total // 3 - 17, 0])
        pool = Pool(256, 400, 5, 200)
        got, want = pool.plan(np.array([5, 0, 255, 256, 9]), add, n)
        _equal(got, want)
        pool.check()


def test_pools_that_are_wrong():
    """Counts past their arrays, and pages that are not: nothing is read or written outside."""
    i32 = dict(dtype=torch.int32, device="cuda")
    guard = torch.full((3, 10), 55, **i32)
    for n_free, held in ((1000, 2), (-5, 1000), (4, -3), (10, 4)):
        free = torch.tensor([3, -1, 99, 2**31 - 1, 5, 6, 7, 8, 9, 1], **i32)
        table = torch.full((3, 4), 77, **i32)
        pool = KvPool(64, free, torch.tensor([n_free], **i32), table, torch.full((3,), held, **i32))
        start, slots, pos, granted = (torch.zeros(k, **i32) for k in (4, 300, 300, 3))
        lens = torch.tensor([0, 64, 200], **i32)
        kv_plan(None, pool, lens, torch.tensor([100, 150, 50], **i32), 300, start, slots, pos, granted)
        kv_release(None, pool, lens)
        kv_release(None, pool, lens * 0)
        torch.cuda.synchronize()
        assert ((slots >= -1) & (slots < 10 * 64)).all()
        assert 0 <= int(pool.n_free) <= 10 and ((pool.held >= 0) & (pool.held <= 4)).all()
        assert (guard == 55).all()


@pytest.mark.parametrize("n", [100, 5000])
def test_graphs(n):
    """A captured round of release and plan follows its arrays from replay to replay."""
    pool, twin = Pool(64, 500, 4, 100), Pool(64, 500, 4, 100)
    lens, add = _dev([0, 0, 0, 0]), _dev([0, 0, 0, 0])
    out = [torch.zeros(k, dtype=torch.int32, device="cuda") for k in (5, n, n, 4)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        kv_release(stream, pool.dev, lens)
        kv_plan(stream, pool.dev, lens, add, n, *out)

    graph = Graph.capture(stream, step)
    for a, m in (([0, 0, 0, 0], [40, 3, 0, 50]), ([40, 0, 0, 50], [1, 64, 5, 0]), ([10, 0, 0, 0], [90, 0, 0, 10])):
        lens.copy_(_dev(a)), add.copy_(_dev(m))
        stream.wait_stream(torch.cuda.current_stream())
        graph.launch(stream)
        stream.synchronize()
        twin.release(np.array(a))
        got, want = twin.plan(np.array(a), np.array(m), n)
        _equal(out, want)
        _equal(got, want)
        assert torch.equal(pool.dev.table, twin.dev.table) and torch.equal(pool.dev.free, twin.dev.free)
