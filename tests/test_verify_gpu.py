"""The verification of drafts on the GPU against a plain walk in 64 bits: whole numbers, all of them equal. Sums differ from the
oracle's by less than 1e-12 of themselves; a case whose u lies that near to a border between two tokens would be unlucky, none is."""

import numpy as np
import pytest
import torch

from qwenny_amd import Graph, TreeStep

pytestmark = pytest.mark.gpu


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _chances(l, temp):
    """p of a row, or None where it has no choice."""
    if np.isnan(l).any() or not np.isfinite(l.max()) or not (temp >= 0 and np.isfinite(temp)):
        return None
    if temp == 0:
        return np.eye(1, len(l), int(np.argmax(l)))[0]
    p = np.exp((l.astype(np.float64) - float(l.max())) / float(np.float32(temp)))
    return p / p.sum()


def _choose(p, u):
    cum = np.cumsum(p)
    at = np.flatnonzero((cum > float(u) * cum[-1]) & (p > 0))
    return int(at[0]) if len(at) else int(np.flatnonzero(p > 0)[-1])


class Case:
    def __init__(self, news, vocab, tree=False, draft=False, seed=0, temps=(0.7, 1.0, 0.0, 1.3), sharp=3.0, page=64):
        rng = np.random.default_rng(seed + vocab)
        self.news, self.vocab, self.page, self.rng = news, vocab, page, rng
        self.n, self.n_seq = sum(news), len(news)
        self.start = np.cumsum([0] + list(news)).astype(np.int32)
        self.len = rng.integers(0, 500, self.n_seq).astype(np.int32)
        self.table = rng.permutation(self.n_seq * 10).reshape(self.n_seq, 10).astype(np.int32)
        self.temp = np.array([temps[b % len(temps)] for b in range(self.n_seq)], np.float32)
        self.logits = (rng.standard_normal((self.n, vocab)) * sharp).astype(np.float32)
        self.u = rng.random((self.n, 2)).astype(np.float32)
        self.tokens = rng.integers(0, vocab, self.n).astype(np.int32)
        self.masks = None
        self.draft = None
        if draft:
            q = np.exp(self.logits * 0.8 + 0.5 * rng.standard_normal(self.logits.shape))
            self.draft = (q / q.sum(-1, keepdims=True)).astype(np.float32)
        parents = [-1] * self.n
        masks = np.zeros(self.n, np.uint64)
        for b, m in enumerate(news):
            a = self.start[b]
            for i in range(m):
                parents[a + i] = (int(rng.integers(max(0, i - 4), i)) if tree else i - 1) if i else -1
                masks[a + i] = (int(masks[a + parents[a + i]]) if i else 0) | 1 << i
                if i and rng.random() < 0.8:  # a draft that its parent's row would choose, or might
                    row = a + parents[a + i]
                    if draft:
                        self.tokens[a + i] = _choose(self.draft[row].astype(np.float64), rng.random())
                    else:
                        p = _chances(self.logits[row], self.temp[b])
                        self.tokens[a + i] = _choose(p, self.u[row, 1] if rng.random() < 0.8 else rng.random())
        self.parents = parents
        if tree:
            self.masks = masks

    def step(self, max_new=None):
        return TreeStep(self.n, _dev(self.start), _dev(self.len), _dev(self.table), max_new or max(max(self.news), 1),
                        None if self.masks is None else _dev(self.masks.view(np.int64)))

    def buffers(self):
        full = lambda k: torch.full((k,), 77, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(next=full(self.n_seq), count=full(self.n_seq), emit=full(self.n), src=full(self.n), dst=full(self.n), new_len=full(self.n_seq))

    def run(self, gemm, step=None, logits=None, draft=None, stream=None, out=None, temp=True):
        out = out or self.buffers()
        gemm.verify(stream, _dev(self.logits) if logits is None else logits, self.vocab, step or self.step(), self.page, _dev(self.tokens),
                    _dev(self.u), temp=_dev(self.temp) if temp else None,
                    draft=_dev(self.draft) if draft is None and self.draft is not None else draft, **out)
        return out

    def want(self):
        w = dict(next=np.full(self.n_seq, -1), count=np.zeros(self.n_seq, int), emit=np.full(self.n, -1), src=np.full(self.n, -1),
                 dst=np.full(self.n, -1), new_len=self.len.astype(int))
        for b, m in enumerate(self.news):
            if not m:
                continue
            a, path, nxt = self.start[b], [0], None
            while nxt is None:
                i = path[-1]
                row = a + i
                p = _chances(self.logits[row], self.temp[b])
                if p is None:
                    nxt = -1
                elif self.draft is not None and i + 1 < m:
                    t = self.tokens[row + 1]
                    q = self.draft[row].astype(np.float64)
                    if 0 <= t < self.vocab and (p[t] == 1 if self.temp[b] == 0 else float(self.u[row, 0]) * q[t] < p[t]):
                        path.append(i + 1)
                    elif self.temp[b] == 0:
                        nxt = int(p.argmax())
                    else:
                        rest = np.maximum(p - q, 0)
                        nxt = _choose(rest if rest.sum() > 0 else p, self.u[row, 1])
                else:
                    y = _choose(p, self.u[row, 1])
                    child = [] if self.draft is not None else [k for k in range(i + 1, m) if self.parents[a + k] == i and self.tokens[a + k] == y]
                    if child:
                        path.append(child[0])
                    else:
                        nxt = y
            slot = lambda k: self.table[b, (self.len[b] + k) // self.page] * self.page + (self.len[b] + k) % self.page  # noqa: E731, B023
            w["next"][b], w["count"][b], w["new_len"][b] = nxt, len(path) - 1, self.len[b] + len(path)
            for k, i in enumerate(path):
                w["emit"][a + k] = self.tokens[a + path[k + 1]] if k + 1 < len(path) else nxt
                if i != k:
                    w["src"][a + k], w["dst"][a + k] = slot(i), slot(k)
        return w

    def check(self, gemm, **kw):
        got, want = self.run(gemm, **kw), self.want()
        for name, w in want.items():
            g = got[name].cpu().numpy()
            assert np.array_equal(g, w), (name, np.flatnonzero(g != w)[:5], g[g != w][:5], w[g != w][:5])
        return want


@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 4095, 4096, 4097, 10007, 70001])
@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
def test_vocabularies(gemm, vocab, kind):
    print(f"{kind} over {vocab}", flush=True)
    Case([5, 1, 3, 4, 2], vocab, tree=kind == "tree", draft=kind == "draft").check(gemm)


@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
@pytest.mark.parametrize("news", [[1], [2], [64], [1] * 64, [0, 3, 0, 0, 5, 0], [64, 1, 33, 17]], ids=str)
def test_sequences(gemm, kind, news):
    print(f"{kind} {news}", flush=True)
    for seed in range(4):
        Case(news, 1000, tree=kind == "tree", draft=kind == "draft", seed=seed, sharp=2.0 + 2 * seed).check(gemm)


@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
def test_a_large_vocabulary(gemm, kind):
    """As flat as logits get, where each token has 4e-6 of the sum, and peaked."""
    for sharp in (0.1, 2.5):
        print(f"{kind} {sharp}", flush=True)
        Case([5, 3, 8], 248320, tree=kind == "tree", draft=kind == "draft", sharp=sharp).check(gemm)


@pytest.mark.parametrize("kind", ["chain", "draft"])
def test_many_sequences(gemm, kind):
    print(f"1024 {kind}", flush=True)
    kept = Case([b % 4 for b in range(1024)], 500, draft=kind == "draft").check(gemm)["count"]
    assert kept.max() >= 2 and (kept == 0).any()


@pytest.mark.parametrize("kind", ["chain", "tree", "draft"])
def test_rows_without_a_choice(gemm, kind):
    """NaN, infinities, rows of nothing and temperatures that are none end a sequence; filtered logits (-inf) are never chosen."""
    c = Case([4] * 9, 5000, tree=kind == "tree", draft=kind == "draft", temps=(0.7, 1.0, 0.0))
    c.logits[0, 4999] = np.nan  # a root's
    c.logits[5, 17] = np.inf
    c.logits[8:12] = -np.inf
    c.logits[12:16, 10:4990] = -np.inf  # whole parts of a row filtered
    c.logits[16:20, :] = -np.inf
    c.logits[16:20, 4321] = -5.0  # one token left
    c.logits[20] = -3e38
    c.temp[6], c.temp[7], c.temp[8] = -1.0, np.nan, np.inf
    c.check(gemm)


@pytest.mark.parametrize("kind", ["chain", "draft"])
def test_ties(gemm, kind):
    """The lowest of equal logits is the likeliest, wherever the equals lie; all logits equal."""
    c = Case([3, 3, 3], 9000, draft=kind == "draft", temps=(0.0, 0.0, 1.0))
    c.logits[:3] = np.minimum(c.logits[:3], 5.0)
    c.logits[:3, [8999, 8191, 4096, 70, 69]] = 6.0
    c.logits[3:] = 0.25
    c.tokens[1], c.tokens[4] = 69, 0
    c.check(gemm)


def test_random_numbers_at_their_ends(gemm):
    """u = 0 is the first token that has any probability, the largest u below 1 the last."""
    for kind in ("chain", "draft"):
        c = Case([2] * 8, 5003, draft=kind == "draft", temps=(1.0,))
        c.logits[:, :7] = -np.inf
        c.logits[:, -9:] = -np.inf
        c.u[:8], c.u[8:] = 0.0, np.nextafter(np.float32(1), np.float32(0))
        if kind == "draft":
            c.draft[:] = 0.0
            c.draft[::2, 100] = 1.0
            c.tokens[1::2] = 100
        c.check(gemm)


def test_tokens_outside_the_vocabulary(gemm):
    for kind in ("chain", "draft"):
        c = Case([3] * 5, 700, draft=kind == "draft")
        c.tokens[[1, 4, 7, 10, 13]] = [-1, 700, 2**31 - 1, -2**31, 5]
        c.check(gemm)


def test_children_that_say_the_same(gemm):
    """Of equal children the first is taken, with what hangs on it."""
    c = Case([5], 50, tree=True, temps=(0.0,))
    c.parents = [-1, 0, 0, 1, 2]
    c.masks = np.array([1, 3, 5, 11, 21], np.uint64)
    first, second = int(c.logits[0].argmax()), int(c.logits[1].argmax())
    c.tokens[:] = [9, first, first, second, int(c.logits[2].argmax())]
    assert c.check(gemm)["count"][0] == 2


def test_trees_of_any_masks(gemm):
    """Masks that are no trees: whatever comes, it lies inside."""
    c = Case([64, 7], 100, tree=True)
    c.masks = c.rng.integers(0, 2**63, c.n).astype(np.uint64)
    got = {k: v.cpu().numpy() for k, v in c.run(gemm).items()}
    assert (got["count"] >= 0).all() and (got["count"] < [64, 7]).all()
    assert (got["emit"] >= -1).all() and (got["emit"] < 100).all()


def test_drafts_of_the_targets_own_probabilities(gemm):
    """Where q is p nothing is rejected but by rounding, and then the choice is p's own; drafts that leave nothing over likewise."""
    c = Case([4, 4], 300, draft=True, temps=(1.0,))
    c.draft[:] = 1.0  # above p everywhere: max(0, p - q) is empty
    c.u[:, 0] = 0.999
    assert (c.check(gemm)["count"] == 0).all()


def test_the_shares_are_the_targets(gemm):
    """Numbers spread evenly over [0, 1) choose each token as often as its probability says, to one number."""
    l = (np.random.default_rng(1).standard_normal(12) * 2).astype(np.float32)
    c = Case([1] * 1024, 12, temps=(1.0,))
    c.logits[:] = l
    c.u[:, 1] = (np.arange(1024) + 0.5) / 1024
    c.check(gemm)
    share = np.bincount(c.run(gemm)["next"].cpu().numpy(), minlength=12) / 1024
    assert (np.abs(share - _chances(l, 1.0)) <= 1 / 1024).all()


def test_strides_and_padding(gemm):
    """Rows of any stride and alignment; tokens behind the last sequence say nothing; no temperatures are temperatures of 1."""
    for kind in ("chain", "draft"):
        c = Case([3, 2, 4], 1001, draft=kind == "draft", temps=(1.0,))
        wide = torch.full((c.n, 1405), float("nan"), device="cuda")
        wide[:, 3:1004] = _dev(c.logits)
        more = torch.full((c.n, 2000), float("nan"), device="cuda")
        if kind == "draft":
            more[:, 1:1002] = _dev(c.draft)
        want = c.want()
        got = c.run(gemm, logits=wide[:, 3:1004], draft=more[:, 1:1002] if kind == "draft" else None, temp=False)
        for name, w in want.items():
            assert np.array_equal(got[name].cpu().numpy(), w), name
    c = Case([3, 2], 300)
    c.logits = np.concatenate((c.logits, np.full((4, 300), np.nan, np.float32)))
    c.tokens, c.u, c.n = np.r_[c.tokens, np.zeros(4, np.int32)], np.concatenate((c.u, np.zeros((4, 2), np.float32))), 9
    c.check(gemm, step=c.step(5))


HUGE = 2**31 - 1


@pytest.mark.parametrize("start,lens,kinds", [([0, 5, 3, 9], None, "x"), ([0, 3, 5, HUGE], None, "==n"), ([-4, 3, 5, 9], None, "n=="),
                                              ([0, 3, 5, 9], [10, -1, 10], "=n="), ([0, 3, 5, 9], [10, HUGE, 637], "=nn"),
                                              ([9, 9, 9, 9], None, "nnn"), ([0, 0, 0, 0], None, "nnn")], ids=str)
def test_numbers_that_do_not_fit(gemm, start, lens, kinds):
    for draft in (False, True):
        c = Case([3, 2, 4], 400, draft=draft)
        if lens:
            c.len[[0, 2]] = 10
        want = c.want()
        c.start = np.array(start, np.int64).astype(np.int32)
        if lens:
            c.len = np.array(lens, np.int64).astype(np.int32)
        got = {k: v.cpu().numpy() for k, v in c.run(gemm).items()}
        if kinds == "x":
            assert got["next"][1] == -1
            continue
        for b, (kind, rows) in enumerate(zip(kinds, (slice(0, 3), slice(3, 5), slice(5, 9)))):
            if kind == "n":
                assert got["next"][b] == -1 and got["count"][b] == 0 and got["new_len"][b] == c.len[b]
                assert all((got[k][rows] == -1).all() for k in ("emit", "src", "dst"))
            else:
                assert got["next"][b] == want["next"][b] and np.array_equal(got["emit"][rows], want["emit"][rows])


@pytest.mark.parametrize("draft", [False, True])
def test_starts_that_go_back_into_a_sequence(gemm, draft):
    """The sequences whose numbers fit keep their own temperatures, whoever else claims their tokens."""
    c = Case([10, 0, 10, 10], 400, draft=draft, temps=(1.3, 0.2, 0.4, 0.8), sharp=1.0)
    if not draft:
        for i in range(1, 10):  # the first sequence's path goes through all of its rows
            c.tokens[i] = _choose(_chances(c.logits[i - 1], c.temp[0]), c.u[i - 1, 1])
    want = c.want()
    c.start = np.array([0, 10, 5, 20, 30], np.int32)
    got = {k: v.cpu().numpy() for k, v in c.run(gemm).items()}
    for b, rows in ((0, slice(0, 10)), (3, slice(20, 30))):
        assert got["next"][b] == want["next"][b] and got["count"][b] == want["count"][b]
        assert np.array_equal(got["emit"][rows], want["emit"][rows])
    assert (got["next"][1:3] == -1).all() and (got["emit"][10:20] == -1).all()


def test_moves_without_tables(gemm):
    """Who wants no moves gives none; pages outside of any cache move nothing."""
    c = Case([4, 5], 300, tree=True)
    want = c.want()
    out = c.buffers()
    out.update(src=None, dst=None, new_len=None)
    got = c.run(gemm, out=out)
    for name in ("next", "count", "emit"):
        assert np.array_equal(got[name].cpu().numpy(), want[name])
    c.table[:] = -1
    got = c.run(gemm)
    assert (got["src"] == -1).all() and (got["dst"] == -1).all()


@pytest.mark.parametrize("kind", ["tree", "draft"])
def test_graphs(gemm, kind):
    """Captured calls on a stream of their own follow their inputs; two of them share the context's scratch."""
    cases = [Case([5, 3, 1], 9001, tree=kind == "tree", draft=kind == "draft", seed=s) for s in range(3)]
    c = cases[0]
    fixed = {k: _dev(getattr(c, k)) for k in ("logits", "tokens", "u", "temp")}
    draft = None if c.draft is None else _dev(c.draft)
    step, outs = c.step(), [c.buffers(), c.buffers()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = [Graph.capture(stream, lambda o=o: gemm.verify(stream, fixed["logits"], c.vocab, step, c.page, fixed["tokens"], fixed["u"],
                                                           temp=fixed["temp"], draft=draft, **o)) for o in outs]
    for other in cases + cases[:1]:
        other.start, other.len, other.table, other.masks, other.parents = c.start, c.len, c.table, c.masks, c.parents
        for k, t in fixed.items():
            t.copy_(_dev(getattr(other, k)))
        if draft is not None:
            draft.copy_(_dev(other.draft))
        stream.wait_stream(torch.cuda.current_stream())
        for g, o in zip(graphs, outs):
            g.launch(stream)
        stream.synchronize()
        want = other.want()
        for o in outs:
            for name, w in want.items():
                assert np.array_equal(o[name].cpu().numpy(), w), name
