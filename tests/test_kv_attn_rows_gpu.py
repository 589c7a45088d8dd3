"""Which rows the attention writes, and what, where a step's numbers do not fit: every row, NaN for the tokens of a sequence that
cannot be served and for no other, zeros for padding."""

import numpy as np
import pytest
import torch

from qwenny_amd import Graph, KvFmt, TreeStep
from tests.test_kv_attn_forms_gpu import Wide
from tests.test_kv_attn_gpu import Step, _dev

pytestmark = pytest.mark.gpu

SEQS = [(100, 2), (300, 3), (4000, 1)]  # the last one's results are joined
HUGE = 2**31 - 1

# starts, max_new -> each row's kind: as with the right starts (=), NaN (n), zeros (0)
STARTS = [([0, 2, 5, 6], 3, "======"), ([0, 5, 5, 6], 3, "nnnnn="), ([0, 2, 2, 6], 3, "==nnnn"), ([0, 70, 5, 6], 3, "nnnnn="),
          ([0, 2, 1, 6], 3, "==nnnn"), ([0, 2, 5, HUGE], 3, "=====n"), ([-5, 2, 5, 6], 3, "nn===="), ([-5, -2, 5, 6], 3, "nnnnn="),
          ([9, 9, 9, 9], 3, "nnnnnn"), ([0, 2, 5, 5], 3, "=====0"), ([2, 2, 5, 6], 3, "00===="), ([0, 0, 0, 0], 3, "000000"),
          ([6, 6, 6, 6], 3, "000000"), ([5, 5, 5, 6], 3, "00000="), ([0, 2, 5, 6], 2, "==nnn="), ([-HUGE - 1, HUGE, -1, HUGE], 3, "nnnnnn")]


def _check(out, clean, kinds):
    for t, kind in enumerate(kinds):
        if kind == "n":
            assert out[t].isnan().all(), t
        else:
            assert torch.equal(out[t], clean[t] if kind == "=" else torch.zeros_like(out[t])), t


@pytest.mark.parametrize("form", [Step, Wide])
@pytest.mark.parametrize("start,max_new,kinds", STARTS, ids=str)
def test_starts(gemm, form, start, max_new, kinds):
    print(f"{form.__name__} {start} up to {max_new}", flush=True)
    s = form(SEQS, KvFmt.I8, 4, 2, 128, 64, gate=True)
    clean = s.run(gemm, step=s.step(3))
    s.check(gemm)
    s.start = np.array(start, np.int64).astype(np.int32)
    _check(s.run(gemm, step=s.step(max_new)), clean, kinds)


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d,tokens", [(64, 1), (256, 5), (128, 40)])
def test_lengths_past_the_table(gemm, fmt, d, tokens):
    """Without the sequences beside them being touched; one that has no tokens may hold any length."""
    seqs = [(300, tokens), (900, tokens), (64, 0), (5000, tokens)]
    for form in (Step, Wide):
        for old in (-1, -HUGE, HUGE, None):
            print(f"{form.__name__} {fmt!r} {d} {tokens} {old}", flush=True)
            s = form(seqs, fmt, 6, 1, d, 64)
            clean = s.run(gemm)
            s.len[1] = s.table.shape[1] * 64 - tokens + 1 if old is None else old
            s.len[2] = old or 0
            _check(s.run(gemm), clean, "=" * tokens + "n" * tokens + "=" * tokens)


@pytest.mark.parametrize("n_seq", [64, 65, 300, 1024])
def test_many_sequences_some_of_which_do_not_fit(gemm, n_seq):
    """The list of more than 64 sequences is made by the workgroup's waves together."""
    print(f"{n_seq} sequences", flush=True)
    s = Step([(b % 70, b % 3) for b in range(n_seq)], KvFmt.E4M3, 2, 1, 64, 64)
    clean, right = s.run(gemm), s.start.copy()
    for change in ("past the end", "descends", "outside"):
        s.start = right.copy()
        kinds = ["="] * s.n
        bad = n_seq - 9  # a sequence before it ends, and it begins, where it should not
        while s.seqs[bad][1] == 0 or s.seqs[bad - 1][1] == 0:
            bad -= 1
        if change == "past the end":
            s.start[bad] = s.n + 7
        elif change == "descends":
            s.start[bad] = right[bad // 2]
        else:
            s.start[0] = -1
        lo, hi = (right[bad - 1], right[bad + 1]) if change != "outside" else (0, right[1])
        kinds[lo:hi] = "n" * (hi - lo)
        print(change, bad, flush=True)
        _check(s.run(gemm), clean, kinds)


def test_replays_that_outgrow_the_capture(gemm):
    """A captured step whose tokens come to be distributed so that one sequence has more than max_new: no row of an earlier
    replay is handed on."""
    s = Wide([(100, 2), (300, 3), (10, 1)], KvFmt.I8, 4, 2, 128, 64)
    start = _dev(s.start)
    step = TreeStep(s.n, start, _dev(s.len), _dev(s.table), 3)
    clean, out, side = s.run(gemm, step=step), torch.zeros((6, 4, 128), dtype=torch.bfloat16, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    g = Graph.capture(side, lambda: gemm.tree_attn(side, s.q, 4, s.kv, step, out))
    for now, kinds in (([0, 2, 5, 6], "======"), ([0, 5, 5, 6], "nnnnn="), ([0, 2, 5, 6], "======"), ([0, 2, 5, 5], "=====0"),
                       ([0, 2, 5, 6], "======")):
        start.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        g.launch(side)
        torch.cuda.synchronize()
        _check(out, clean, kinds)
