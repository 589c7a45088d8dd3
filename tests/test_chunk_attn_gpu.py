"""The attention of prompt chunks over the cache against a plain form in 64 bits: lengths from one token on, head layouts, ragged
batches, what the rows do not see, rows of sequences that do not fit, graphs and streams. Tolerances as in the step's attention:
half a step of bf16 is 2^-8 of the value, of f16 2^-11, of f32 2^-24."""

import numpy as np
import pytest
import torch

from qwenny_amd import Graph, KvCache, KvFmt, TreeStep, kv_write
from tests.test_kv_attn_gpu import TOP, Host, Step, _dev, _f64

pytestmark = pytest.mark.gpu


class Chunk(Step):
    """Sequences (cached, new) whose new tokens are chunks: each sees all positions before it, and its own."""

    def run(self, gemm, scale=None, step=None, stream=None):
        out = torch.full((self.n, self.h, self.d), 77.0, dtype=torch.bfloat16, device="cuda")
        gemm.chunk_attn(stream, self.q, self.h, self.kv, step or self.step(), out, gate=self.gate, scale=scale)
        return out

    def want(self, scale=None):
        scale = self.d**-0.5 if scale is None else scale
        host, g = Host(self.kv), self.h // self.j
        out, tol = np.zeros((2, self.n, self.h, self.d))
        q = _f64(self.q)
        for b, (a, m) in enumerate(self.seqs):
            kv, scales = host.values(self.slots[b]), host.scales[self.slots[b]].astype(np.float64)
            late = np.arange(a + m) > a + np.arange(m)[:, None]
            for head in range(self.h) if m else ():
                mine = slice(self.start[b], self.start[b + 1])
                k, v, vs = kv[:, head // g, 0], kv[:, head // g, 1], scales[:, head // g, 1]
                s = np.where(late, -np.inf, q[mine, head] @ k.T * scale)
                top = s.max(-1, keepdims=True)
                p = np.exp(s - top)
                l = p.sum(-1, keepdims=True)
                out[mine, head] = p @ v / l
                # scores: sums of d products in f32, then two products; of the exponent's argument (in units of log 2) one rounding;
                # the exponential a few units in the last place
                ds = np.where(late, 0, np.abs(q[mine, head]) @ np.abs(k).T * scale * (self.d + 8) * 2.0**-24).max(-1, keepdims=True)
                ds += np.where(late, 0, top - s).max(-1, keepdims=True) * 2.0**-22
                seen = a + np.arange(m)[:, None] + 1
                # a probability is rounded to f16, and so are a value's scale and the value: 2^-11 of it each (where a row does not see all of
                # a tile, only the probability times the scale is); or half of f16's smallest step relative to the largest scale that
                # the row sees (the reference is at most twice that)
                small = seen * 2.0**-25 * 2 * np.where(late, 0, np.abs(vs)).max(-1, keepdims=True) * TOP[self.kv.fmt] / l
                tol[mine, head] = (3 * 2.0**-11 + 4 * ds + (seen + 64) * 2.0**-23) * (p @ np.abs(v) / l) + small
        if self.gate is not None:
            sig = 1 / (1 + np.exp(-_f64(self.gate)))
            out, tol = out * sig, tol * sig + np.abs(out * sig) * 2.0**-20
        return out, tol + np.abs(out) * 2.0**-8 + 1e-38

    def check_rows(self, got, rows, scale=None):
        out, tol = self.want(scale)
        off = np.abs(_f64(got) - out) - tol
        assert np.isfinite(_f64(got)[rows]).all()
        assert (off[rows] <= 0).all(), off[rows].max()


class Wide(Chunk):
    """The same with tables of far more positions than the sequences have: units of twice the rows, shared in parts where that is
    worth it."""

    def step(self, max_new=None):
        if self.table.shape[1] * self.kv.page < 90 * 64:
            more = -(-90 * 64 // self.kv.page) - self.table.shape[1]
            self.table = np.concatenate((self.table, np.full((len(self.seqs), more), -7, np.int32)), 1)
        return super().step(max_new)


FORMS = pytest.mark.parametrize("form", [Chunk, Wide])
SHORT = [[(0, 1)], [(0, 2)], [(0, 31)], [(0, 32)], [(0, 33)], [(0, 64)], [(0, 65)], [(1, 64)], [(63, 1)], [(63, 2)], [(64, 130)], [(100, 257)],
         [(1000, 43)], [(511, 86)]]


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("seqs", SHORT, ids=str)
def test_short_lengths(gemm, form, fmt, seqs):
    print(f"chunk {fmt!r} {seqs}", flush=True)
    form(seqs, fmt, 6, 1, 256, 64, gate=True).check(gemm)


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,j,page", [(1, 1, 64), (4, 4, 128), (16, 4, 256), (7, 1, 1024), (17, 1, 64), (64, 1, 64)])
def test_head_layouts(gemm, form, fmt, d, h, j, page):
    print(f"chunk {fmt!r} {h}/{j}x{d} page {page}", flush=True)
    form([(300, 70), (0, 3)], fmt, h, j, d, page, seed=h).check(gemm)


RAGGED = [(50, 100), (0, 0), (4, 1), (0, 200), (129, 64), (3, 0), (700, 31), (2000, 1), (63, 65)]


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d,h,j", [(256, 24, 4), (128, 8, 8), (64, 4, 1)])
def test_ragged_batches(gemm, form, fmt, d, h, j):
    print(f"chunks {fmt!r} {h}/{j}x{d}", flush=True)
    form(RAGGED, fmt, h, j, d, 128).check(gemm)


@FORMS
def test_many_sequences(gemm, form):
    """As many sequences as a step takes: the plan's last places."""
    print("1024 sequences", flush=True)
    form([(b % 70, b % 3 if b % 100 else 80) for b in range(1024)], KvFmt.I8, 2, 1, 64, 64).check(gemm)


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("written", [False, True])
@pytest.mark.parametrize("seqs", [[(16, 5)], [(300, 70), (0, 3), (1000, 130)]], ids=str)
def test_negative_scales(gemm, form, fmt, written, seqs):
    """Where nothing was written the cache may hold any; where a program wrote its own codes, scales of either sign."""
    s = form(seqs, fmt, 8, 2, 128, 64, gate=True)
    held = s.kv.scales.clone()
    sign = torch.where(torch.rand(held.shape, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0).cuda()
    if written:
        s.kv.scales.copy_(held * sign)
    else:
        scales = Host(s.kv).scales
        s.kv.scales.copy_(torch.where(torch.isfinite(held) & (held < 1e38), held, sign * 0.37))
        every = np.concatenate(s.slots)
        assert np.array_equal(Host(s.kv).scales[every], scales[every])
    s.check(gemm)


@pytest.mark.parametrize("fmt,seqs,h,j,d", [(KvFmt.I8, [(20001, 66)], 6, 1, 256), (KvFmt.E4M3, [(9000, 90)], 12, 2, 128),
                                            (KvFmt.E4M3, [(30000, 65)], 2, 1, 64), (KvFmt.I8, [(5000, 300), (7, 80)], 6, 2, 256)], ids=str)
def test_long_caches(gemm, fmt, seqs, h, j, d):
    print(f"long {fmt!r} {seqs} {h}/{j}x{d}", flush=True)
    s = Chunk(seqs, fmt, h, j, d, 256, gate=True)
    s.check(gemm)
    assert torch.equal(s.run(gemm), s.run(gemm))


@FORMS
@pytest.mark.parametrize("scale", [1.0, 1e-4, 30.0])
@pytest.mark.parametrize("fmt", list(KvFmt))
def test_scales(gemm, form, fmt, scale):
    """A flat softmax, and one so peaked that all but one probability vanish."""
    form([(700, 70)], fmt, 4, 2, 128, 64).check(gemm, scale=scale)


def test_max_new_above_what_is_there(gemm):
    s = Chunk([(100, 70), (50, 1)], KvFmt.I8, 4, 2, 128, 64)
    s.check(gemm, step=s.step(5000))


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("rising", [True, False])
def test_values_of_very_different_size(gemm, form, fmt, d, rising):
    """Over 2^100 from the first position to the last and back: what a row sees later is taken relative to a larger scale."""
    s = form([(500, 200), (0, 70)], fmt, 4, 2, d, 64, gate=True)
    for slots in s.slots:
        at = np.arange(len(slots)) / len(slots)
        size = 2.0 ** (100 * (at if rising else 1 - at) - 60)
        v = _dev(s.rng.standard_normal((len(slots), 2, d)) * size[:, None, None], torch.bfloat16)
        k = _dev(s.rng.standard_normal((len(slots), 2, d)), torch.bfloat16)
        kv_write(None, s.kv, k, v, _dev(slots.astype(np.int32)), len(slots))
    s.check(gemm)


@FORMS
@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("which", [0, 1])
def test_what_a_row_does_not_see(gemm, form, fmt, bad, which):
    """A later token's key or value that is not finite, or huge, and what lies behind the sequence's end, take nothing from a row
    before it; rows from it on have it."""
    s = form([(100, 90), (0, 70)], fmt, 4, 2, 128, 64)
    out, tol = s.want()
    at = 140  # a token of the first sequence: its 40th new one
    for head in range(2):  # the last entry is what follows the sequence
        for slot in (s.slots[0][at], s.slots[0][-1] // 64 * 64 + 63):  # (written twice: the second kv head's stays bad)
            kv = [s.k[at:at + 1].clone(), s.v[at:at + 1].clone()]
            kv[which][0, head, 5] = bad
            kv_write(None, s.kv, kv[0], kv[1], _dev(np.array([slot], np.int32)), 1)
    got = s.run(gemm)
    clean = np.r_[0:40, 90:160]
    off = np.abs(_f64(got) - out) - tol
    assert (off[clean] <= 0).all(), off[clean].max()
    assert (off[40:90, :2] <= 0).all(), off[40:90, :2].max()
    if bad != 3e38:
        assert torch.isnan(got[40:90, 2:]).all()
    elif which:
        s.check_rows(got, np.r_[0:160])


@FORMS
def test_queries_that_are_not_finite(gemm, form):
    s = form([(100, 90)], KvFmt.I8, 4, 2, 128, 64)
    s.q[3, 1, 7] = float("nan")
    s.q[70, 2, 100] = float("inf")
    s.q[5, 0] = 0.0
    s.q[6, 0, 3] = 3e38
    got = s.run(gemm)
    assert torch.isnan(got[3, 1]).all() and torch.isnan(got[70, 2]).all()
    s.q[3, 1], s.q[70, 2] = 0.0, 0.0
    out, tol = s.want()
    off = np.abs(_f64(got) - out) - tol
    off[3, 1] = off[70, 2] = 0
    assert (off <= 0).all(), off.max()


@FORMS
def test_pages_outside_the_cache(gemm, form):
    s = form([(100, 90), (200, 70)], KvFmt.E4M3, 4, 2, 128, 64)
    out, tol = s.want()
    for page in (-1, s.kv.pages, 2**31 - 1):
        s.table[0, 2] = page  # positions 128 to 191: tokens from the 28th on
        got = s.run(gemm)
        off = np.abs(_f64(got) - out) - tol
        assert torch.isnan(got[28:90]).all()
        assert (off[np.r_[0:28, 90:160]] <= 0).all()


HUGE = 2**31 - 1
# starts, max_new -> each sequence's kind: as with the right starts (=), NaN (n), zeros (0), of sequences of 70, 3 and 100 tokens
STARTS = [([0, 70, 73, 173], 100, "==="), ([0, 70, 70, 170], 200, "=N"), ([0, 70, 73, HUGE], 100, "==n"), ([-5, 70, 73, 173], 100, "n=="),
          ([0, 70, 73, 73], 100, "==0"), ([0, 0, 0, 0], 100, "000"), ([173, 173, 173, 173], 100, "000"), ([0, 70, 73, 173], 99, "==n"),
          ([0, 70, 73, 173], 60, "n=n"), ([0, 99, 73, 173], 100, None), ([-HUGE - 1, HUGE, -1, HUGE], 100, "nnn")]


@FORMS
@pytest.mark.parametrize("start,max_new,kinds", STARTS, ids=str)
def test_starts(gemm, form, start, max_new, kinds):
    print(f"starts {start} up to {max_new}", flush=True)
    s = form([(100, 70), (300, 3), (40, 100)], KvFmt.I8, 4, 2, 128, 64, gate=True)
    out, tol = s.want()
    s.start = np.array(start, np.int64).astype(np.int32)
    got = s.run(gemm, step=s.step(max_new))
    assert not (got == 77.0).all(-1).any()  # every row is written
    if kinds is None:
        assert torch.isnan(got[73:99]).all()
        return
    for kind, rows in zip(kinds, (slice(0, 70), slice(70, 73), slice(73, 173))):
        if kind == "N":  # the two after it have one start: all tokens are the last one's, which is served as other positions
            assert torch.isfinite(got[70:170]).all() and (got[170:] == 0).all()
            continue
        if kind == "n":
            assert torch.isnan(got[rows]).all()
        elif kind == "0":
            assert (got[rows] == 0).all()
        else:
            assert (np.abs(_f64(got)[rows] - out[rows]) <= tol[rows]).all()


@FORMS
@pytest.mark.parametrize("old", [-1, -HUGE, HUGE, None])
def test_lengths_past_the_table(gemm, form, old):
    s = form([(300, 70), (900, 66), (64, 0), (700, 80)], KvFmt.I8, 6, 1, 64, 64)
    out, tol = s.want()
    s.len[1] = s.table.shape[1] * 64 - 65 if old is None else old
    s.len[2] = old or 0
    got = s.run(gemm)
    rows = np.r_[0:70, 136:216]
    assert torch.isnan(got[70:136]).all() and (np.abs(_f64(got)[rows] - out[rows]) <= tol[rows]).all()


def test_padding_and_strides_of_tables(gemm):
    """Tokens behind the last sequence are zeros; tables wider than the sequences need."""
    s = Chunk([(300, 70), (20, 10)], KvFmt.E4M3, 4, 2, 256, 64)
    n = s.n
    s.q = torch.cat((s.q, torch.full_like(s.q[:13], float("nan"))))
    s.n = n + 13
    s.table = np.concatenate((s.table, np.full((2, 500), 9, np.int32)), 1)
    got = s.run(gemm, step=s.step(200))
    assert (got[n:] == 0).all()
    s.n, s.q = n, s.q[:n]
    s.check_rows(got[:n], np.r_[0:n])


@FORMS
def test_agrees_with_tree_attn(gemm, form):
    """Chains of up to 64 tokens by either operator, each within its bound."""
    s = form([(100, 64), (2000, 1), (0, 30)], KvFmt.I8, 24, 4, 256, 256, gate=True)
    a, b = s.run(gemm), Step.run(s, gemm)
    out, tol = s.want()
    for got in (a, b):
        assert (np.abs(_f64(got) - out) <= tol).all()


def test_far_pages(gemm):
    """Codes past 32-bit offsets: the cache's last pages, beyond 4 GiB."""
    print("far pages", flush=True)
    pages = (5 << 30) // (4 * 2 * 256 * 1024)
    s = FarChunk([(3000, 70)], KvFmt.I8, 8, 4, 256, 1024, first_page=pages - 6, pages=pages)
    s.check(gemm)


class FarChunk(Chunk):
    """A cache too large to look at whole: the host's copy holds its last pages."""

    def want(self, scale=None):
        last, whole, slots = 6, self.kv, self.slots
        self.kv = KvCache(whole.fmt, whole.heads, whole.head_dim, whole.page, whole.codes[-last:], whole.scales[-last:])
        self.slots = [s - (whole.pages - last) * whole.page for s in slots]
        try:
            return super().want(scale)
        finally:
            self.kv, self.slots = whole, slots


@FORMS
@pytest.mark.parametrize("seqs", [[(100, 70)], [(3000, 130), (0, 66), (50, 1)]], ids=str)
def test_graphs(gemm, form, seqs):
    """A captured call follows the lengths and tables from replay to replay; two graphs share the context's scratch."""
    s = form(seqs, KvFmt.I8, 6, 2, 128, 64, gate=True)
    s.step()  # (the form's tables)
    lens = _dev(s.len)
    step = TreeStep(s.n, _dev(s.start), lens, _dev(s.table), max(m for _, m in seqs))
    out = [torch.zeros((s.n, s.h, s.d), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    calls = [lambda o=o: gemm.chunk_attn(stream, s.q, s.h, s.kv, step, o, gate=s.gate) for o in out]
    graphs = [Graph.capture(stream, call) for call in calls]
    for back in (0, 17, 60, 0):
        lens.copy_(_dev(np.maximum(s.len - back, 0)))
        stream.wait_stream(torch.cuda.current_stream())
        for g, o in zip(graphs, out):
            with torch.cuda.stream(stream):
                o.fill_(7)
            g.launch(stream)
        stream.synchronize()
        eager = s.run(gemm, step=step)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager) and torch.equal(out[1], eager)
    out, tol = s.want()
    assert (np.abs(_f64(eager) - out) <= tol).all()
