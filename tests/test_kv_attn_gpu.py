"""The decode step's attention on the GPU against plain forms in 64 bits: the cache's codes bit for bit, attn_prep, the
attention of chains and trees over it, and the operators together. Tolerances count each rounding: half a step of bf16 is
2^-8 of the value, of f16 2^-11, of f32 2^-24."""

import numpy as np
import pytest
import torch

from qwenny_amd import AttnRows, Graph, KvCache, KvFmt, TreeStep, attn_prep, kv_move, kv_read, kv_write

pytestmark = pytest.mark.gpu

TOP = {KvFmt.I8: 127.0, KvFmt.E4M3: 448.0}
E4M3 = np.array([np.nan if c & 127 == 127 else (-1.0) ** (c >> 7) *
                 ((c & 7) * 2.0**-9 if not c >> 3 & 15 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3 & 15) - 7)) for c in range(256)])


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _f64(t):
    return t.detach().cpu().double().numpy()


def _bf16(a):
    """f64 rounded to bf16 through the f32 that holds it (values here are f32 products)."""
    return torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16).double().numpy()


def code_places(d, page):
    """[page][d] -> place in the keys' and in the values' block, as include/qwenny_hip.h says."""
    t, i = np.arange(page)[:, None], np.arange(d)[None]
    return (t // 16 * 16 * d + i // 64 * 1024 + t % 16 * 64 + i % 64,
            t // 64 * 64 * d + i * 64 + t % 16 // 4 * 16 + t % 64 // 16 * 4 + t % 4)


class Host:
    """A cache's contents by slot: codes u8 [slots][heads][2][d] and scales f32 [slots][heads][2]."""

    def __init__(self, kv):
        c = kv.codes.cpu().numpy().reshape(kv.pages, kv.heads, 2, -1)
        k, v = code_places(kv.head_dim, kv.page)
        both = np.stack([c[:, :, 0][..., k], c[:, :, 1][..., v]], 3)  # [pages][heads][page][2][d]
        self.codes = both.transpose(0, 2, 1, 3, 4).reshape(kv.pages * kv.page, kv.heads, 2, kv.head_dim)
        s = kv.scales.cpu().numpy().reshape(kv.pages, kv.heads, 2, kv.page)
        self.scales = s.transpose(0, 3, 1, 2).reshape(kv.pages * kv.page, kv.heads, 2)
        self.fmt = kv.fmt

    def units(self, slots):
        c = self.codes[slots]
        return c.astype(np.float64) - 128 if self.fmt == KvFmt.I8 else E4M3[c]

    def values(self, slots):
        return self.units(slots) * self.scales[slots].astype(np.float64)[..., None]


def quantised(x, fmt):
    """f64 [.., d] of f32 values -> (codes, f32 scales): each code the nearest to x / scale, ties to even."""
    s = (np.abs(x).max(-1) / TOP[fmt]).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        u = np.where(s[..., None] > 0, x / s.astype(np.float64)[..., None], 0.0)
    if fmt == KvFmt.I8:
        return (np.clip(np.rint(u), -127, 127) + 128).astype(np.uint8), s
    unit = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(u), 2.0**-6))) - 3)
    u = np.clip(np.rint(u / unit) * unit, -448, 448)
    table = {E4M3[c]: c for c in range(127)}
    mag = np.vectorize(table.__getitem__, otypes=[np.uint8])(np.abs(u))
    return np.where(np.signbit(u), mag | 128, mag).astype(np.uint8), s


def new_cache(fmt, heads, d, page, pages, seed=0):
    """A cache of what memory may hold: every byte value (e4m3's NaN among them), scales NaN, infinite and huge."""
    kv = KvCache.new(fmt, heads, d, page, pages)
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv.codes.random_(0, 256, generator=g)
    kv.codes.view(-1)[::7] = 127
    kv.scales.fill_(float("nan"))
    kv.scales.view(-1)[1::5] = float("inf")
    kv.scales.view(-1)[2::5] = 3e38
    return kv


# ---- the cache ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("heads,d,page,n", [(1, 64, 64, 1), (4, 256, 256, 37), (2, 128, 64, 300), (8, 64, 1024, 9), (3, 256, 128, 65)])
def test_write_and_read(fmt, heads, d, page, n):
    print(f"cache {fmt!r} {heads}x{d} page {page} n={n}", flush=True)
    rng = np.random.default_rng(n + d)
    pages = -(-2 * n // page) + 1
    kv = new_cache(fmt, heads, d, page, pages)
    before = Host(kv)
    slots = rng.permutation(pages * page)[:n].astype(np.int32)
    if n > 30:  # runs of neighbours, as a prompt's
        slots[4:24] = np.setdiff1d(np.arange(pages * page), np.r_[slots[:4], slots[24:]])[:20]
    x = _dev(rng.standard_normal((2, n, heads, d)) * rng.choice([1e-6, 1.0, 300.0], (2, n, heads, 1)), torch.bfloat16)
    if n > 8:
        x[0, 1] = 0.0
        x[1, 2, 0] = 1.0  # every value the largest
        x[0, 3, 0, :2] = torch.tensor([127.0, 63.5])  # i8: scale 1, a code on a border
        x[0, 4, 0] = torch.finfo(torch.float32).tiny * torch.arange(d).cuda() / d  # scales below the normal numbers
        x[0, 5, 0, 3] = 3e38
    kv_write(None, kv, x[0], x[1], _dev(slots), n)
    after = Host(kv)
    want = _f64(x).transpose(1, 2, 0, 3)  # [n][heads][2][d]
    codes, scales = quantised(want, fmt)
    normal = scales.astype(np.float64) >= 2.0**-126  # a scale below: few bits, the quotient is clamped
    assert np.array_equal(after.scales[slots], scales)
    assert np.array_equal(after.codes[slots][normal], codes[normal])
    rest = np.setdiff1d(np.arange(pages * page), slots)
    assert np.array_equal(after.codes[rest], before.codes[rest])
    assert np.array_equal(after.scales[rest], before.scales[rest], equal_nan=True)
    k, v = torch.full_like(x, float("nan"))
    kv_read(None, kv, _dev(slots), n, k, v)
    back = np.stack([_f64(k), _f64(v)], 2)
    exact = (after.units(slots).astype(np.float32) * after.scales[slots][..., None]).astype(np.float64)
    assert np.array_equal(back, _bf16(exact))


def test_slots_outside_the_cache():
    kv = new_cache(KvFmt.I8, 2, 64, 64, 3)
    before = Host(kv)
    slots = np.array([-1, 5, 3 * 64, 2**31 - 1, -2**31, 191], np.int32)
    x = torch.ones((2, 6, 2, 64), dtype=torch.bfloat16, device="cuda")
    kv_write(None, kv, x[0], x[1], _dev(slots), 6)
    after = Host(kv)
    rest = np.setdiff1d(np.arange(192), [5, 191])
    assert np.array_equal(after.codes[rest], before.codes[rest]) and (after.codes[[5, 191]] == 255).all()
    k, v = torch.full_like(x, float("nan"))
    kv_read(None, kv, _dev(slots), 6, k, v)
    for t in (k, v):
        assert (t[[0, 2, 3, 4]] == 0).all() and (t[[1, 5]] == 1).all()
    src, dst = np.array([5, -1, 7, 192], np.int32), np.array([400, 9, -3, 10], np.int32)
    kv_move(None, kv, _dev(src), _dev(dst), _dev(np.array([0, 4], np.int32)), 1)
    assert np.array_equal(Host(kv).codes, after.codes)


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite(fmt, bad):
    kv = new_cache(fmt, 1, 128, 64, 1)
    x = torch.randn((2, 3, 1, 128), device="cuda").to(torch.bfloat16)
    x[0, 1, 0, 7] = bad
    kv_write(None, kv, x[0], x[1], _dev(np.arange(3, dtype=np.int32)), 3)
    h = Host(kv)
    assert np.isnan(h.scales[1, 0, 0]) and np.isfinite(np.delete(h.scales[:3].reshape(-1), 2)).all()
    assert np.isfinite(h.units(slice(0, 3))).all()
    k, v = torch.empty_like(x)
    kv_read(None, kv, _dev(np.arange(3, dtype=np.int32)), 3, k, v)
    assert k[1].isnan().all() and k[[0, 2]].isfinite().all() and v.isfinite().all()


@pytest.mark.parametrize("d,page", [(64, 64), (128, 128), (256, 256)])
def test_move(d, page):
    """Ascending paths over their own destinations, more than 64 moves, several sequences, moves onto themselves."""
    print(f"move {d} {page}", flush=True)
    rng = np.random.default_rng(d)
    kv = KvCache.new(KvFmt.E4M3, 3, d, page, 4 * 256 // page + 2)
    kv.codes.random_(0, 256)
    kv.scales.normal_()
    before = Host(kv)
    src, dst, start = [], [], [0]
    for at, m in ((0, 9), (100, 0), (200, 1), (300, 90), (700, 64)):
        path = np.sort(rng.choice(200 if m > 64 else 2 * m + 1, m, replace=False))
        src += list(at + path)
        dst += list(at + np.arange(m))
        start.append(len(src))
    kv_move(None, kv, _dev(np.array(src, np.int32)), _dev(np.array(dst, np.int32)), _dev(np.array(start, np.int32)), 5)
    after = Host(kv)
    want_c, want_s = before.codes.copy(), before.scales.copy()
    want_c[dst], want_s[dst] = before.codes[src], before.scales[src]
    assert np.array_equal(after.codes, want_c) and np.array_equal(after.scales, want_s)


# ---- attn_prep ------------------------------------------------------------------------------------------------------


def prep_f64(x, q_heads, kv_heads, d, rot, gated, q_w, k_w, inv_freq, pos, eps):
    """(q, gate, k, v) of partials x [splits][n][rows] in f64, and bounds of the values that went into each: [n][heads][d]."""
    s, n, rows = x.shape
    u, m = x.sum(0).reshape(n, -1, d), np.abs(x).sum(0).reshape(n, -1, d)
    nq = q_heads * (2 if gated else 1)
    step = 2 if gated else 1

    def head(lo, hi, by, w):
        y, b = u[:, lo:hi:by], m[:, lo:hi:by]
        if w is not None:
            r = 1 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
            y, b = y * r * w, b * r * np.abs(w)
        if rot:
            a = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
            c, si = np.cos(a)[:, None], np.sin(a)[:, None]
            h = rot // 2
            y = np.concatenate([y[..., :h] * c - y[..., h:rot] * si, y[..., h:rot] * c + y[..., :h] * si, y[..., rot:]], -1)
            both = b[..., :h] + b[..., h:rot]
            b = np.concatenate([both, both, b[..., rot:]], -1)
        return y, b

    plain = lambda lo, hi, by: (u[:, lo:hi:by], m[:, lo:hi:by])  # noqa: E731
    return (head(0, nq, step, q_w), plain(1, nq, 2) if gated else None, head(nq, nq + kv_heads, 1, k_w),
            plain(nq + kv_heads, nq + 2 * kv_heads, 1))


# q heads, kv heads, d, rot, gated, splits, n, norm
PREPS = [(16, 4, 256, 64, True, 8, 1, True), (24, 4, 256, 64, True, 3, 5, True), (6, 2, 128, 128, False, 1, 33, True),
         (4, 4, 64, 16, True, 11, 2, False), (3, 1, 128, 0, False, 2, 7, True), (2, 1, 256, 256, False, 1, 600, True),
         (5, 5, 64, 6, False, 1, 3, True), (1, 1, 64, 64, True, 20, 1, True)]


def _prep_inputs(h, j, d, rot, gated, splits, n):
    rng = np.random.default_rng(h * 1000 + n)
    rows = AttnRows(h, j, d, rot, gated)
    x = (rng.standard_normal((splits, n, rows.rows)) * 2).astype(np.float32)
    q_w, k_w = rng.uniform(0.5, 1.5, (2, d)).astype(np.float32)
    inv_freq = (1e7 ** (-np.arange(rot // 2) / max(1, rot // 2))).astype(np.float32)
    pos = rng.integers(0, 262144, n).astype(np.int32)
    pos[0] = 2**31 - 1 if n > 2 else pos[0]  # the angle is exact at any position
    return rows, x, q_w, k_w, inv_freq, pos


def _prep_tol(bound, splits, d):
    # f32: the partials' sum, the mean of squares (d terms, its error halved by the root), a few products; the sine and
    # cosine and their fraction of a turn are good to 2^-22
    return bound * (splits + d / 2 + 40) * 2.0**-24


@pytest.mark.parametrize("h,j,d,rot,gated,splits,n,norm", PREPS)
def test_prep_dense(h, j, d, rot, gated, splits, n, norm):
    print(f"prep {h}/{j}x{d} rot {rot} gated {gated} splits {splits} n={n}", flush=True)
    rows, x, q_w, k_w, inv_freq, pos = _prep_inputs(h, j, d, rot, gated, splits, n)
    bf = lambda heads: torch.full((n, heads, d), float("nan"), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, gate, k, v = bf(h), bf(h) if gated else None, bf(j), bf(j)
    attn_prep(None, _dev(x), splits, n, rows, _dev(q_w) if norm else None, _dev(k_w) if norm else None, _dev(inv_freq), _dev(pos), q,
              gate, k=k, v=v, eps=1e-6)
    want = prep_f64(x.astype(np.float64), h, j, d, rot, gated, q_w if norm else None, k_w if norm else None, inv_freq, pos, 1e-6)
    for name, got, w in zip("qgkv", (q, gate, k, v), want):
        if got is None:
            continue
        y, bound = w
        off = np.abs(_f64(got) - y)
        assert (off <= 2.0**-8 * np.abs(y) + _prep_tol(bound, splits, d)).all(), (name, off.max())


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("h,j,d,rot,gated,splits,n,norm", [PREPS[0], PREPS[1], PREPS[2], PREPS[3], PREPS[5]])
def test_prep_into_the_cache(fmt, h, j, d, rot, gated, splits, n, norm):
    print(f"prep {fmt!r} {h}/{j}x{d} n={n}", flush=True)
    rows, x, q_w, k_w, inv_freq, pos = _prep_inputs(h, j, d, rot, gated, splits, n)
    q, q2, k, v = (torch.empty((n, m, d), dtype=torch.bfloat16, device="cuda") for m in (h, h, j, j))
    gate = torch.empty_like(q) if gated else None
    kv = new_cache(fmt, j, d, 64, n // 64 + 2)
    slots = np.random.default_rng(n).permutation(kv.pages * 64)[:n].astype(np.int32)
    ws = (_dev(q_w), _dev(k_w)) if norm else (None, None)
    attn_prep(None, _dev(x), splits, n, rows, *ws, _dev(inv_freq), _dev(pos), q, gate, kv=kv, slots=_dev(slots))
    attn_prep(None, _dev(x), splits, n, rows, *ws, _dev(inv_freq), _dev(pos), q2, gate, k=k, v=v)
    assert torch.equal(q, q2)
    host = Host(kv)
    want = prep_f64(x.astype(np.float64), h, j, d, rot, gated, q_w if norm else None, k_w if norm else None, inv_freq, pos, 1e-6)
    for which, (y, bound) in enumerate(want[2:]):
        tol = _prep_tol(bound, splits, d)
        units, scale = host.units(slots)[:, :, which], host.scales[slots][:, :, which].astype(np.float64)[..., None]
        top = np.abs(y).max(-1, keepdims=True)
        assert (np.abs(scale * TOP[fmt] - top) <= 2.0**-23 * top + tol.max(-1, keepdims=True)).all()
        # half a step of the code the value lies at; the value over the scale is off by tol / scale and by the scale's error
        u = np.abs(y) / scale
        step = 1.0 if fmt == KvFmt.I8 else 2.0 ** (np.floor(np.log2(np.maximum(u * (1 + 2.0**-10), 2.0**-6))) - 3)
        assert (np.abs(units - y / scale) <= 0.5 * step + tol / scale + 2.0**-22 * u + tol.max(-1, keepdims=True) / scale).all()


# ---- the attention --------------------------------------------------------------------------------------------------


class Step:
    """Sequences (cached, new) over a cache of pages in any order, their inputs, and the attention in f64."""

    def __init__(self, seqs, fmt, h, j, d, page, mask="chain", gate=False, seed=0, q_scale=1.5, first_page=0, pages=None):
        rng = np.random.default_rng(seed + d + h)
        self.seqs, self.h, self.j, self.d, self.rng = seqs, h, j, d, rng
        held = [-(-(a + m) // page) for a, m in seqs]
        count = sum(held) + 2
        self.kv = new_cache(fmt, j, d, page, pages or count + first_page, seed)
        order = list(first_page + rng.permutation(count))
        width = max(held + [1]) + 1
        self.table = np.full((len(seqs), width), -7, np.int32)  # what is past a sequence's pages is never looked at
        for b, m in enumerate(held):
            self.table[b, :m] = [order.pop() for _ in range(m)]
        self.slots = [self.table[b][np.arange(a + m) // page].astype(np.int64) * page + np.arange(a + m) % page
                      for b, (a, m) in enumerate(seqs)]
        every = np.concatenate(self.slots + [np.zeros(0, np.int64)]).astype(np.int32)
        self.k, self.v = (_dev(rng.standard_normal((len(every), j, d)) * rng.choice([0.01, 1.0, 30.0], (len(every), j, 1),
                                                                                    p=[0.1, 0.8, 0.1]), torch.bfloat16) for _ in range(2))
        self.every = _dev(every)
        if len(every):
            kv_write(None, self.kv, self.k, self.v, self.every, len(every))
        self.n = sum(m for _, m in seqs)
        self.start = np.cumsum([0] + [m for _, m in seqs]).astype(np.int32)
        self.len = np.array([a for a, _ in seqs], np.int32)
        self.mask = None
        if mask != "chain":
            self.mask = np.zeros(self.n, np.uint64)
            for b, (a, m) in enumerate(seqs):
                bits = []
                for i in range(m):
                    p = int(rng.integers(-1, i)) if i else -1
                    bits.append((bits[p] if p >= 0 else 0) | 1 << i)
                    if mask == "any":
                        bits[i] = int(rng.integers(0, 2**63)) & int(rng.integers(0, 2**63))
                    if mask == "none":
                        bits[i] = 0
                self.mask[self.start[b]:self.start[b + 1]] = bits
        self.q = _dev(rng.standard_normal((self.n, h, d)) * q_scale * rng.choice([0.05, 1.0], (self.n, h, 1)), torch.bfloat16)
        self.gate = _dev(rng.standard_normal((self.n, h, d)) * 3, torch.bfloat16) if gate else None

    def step(self, max_new=None):
        return TreeStep(self.n, _dev(self.start), _dev(self.len), _dev(self.table), max_new or max([m for _, m in self.seqs] + [1]),
                        None if self.mask is None else _dev(self.mask.view(np.int64)))

    def run(self, gemm, scale=None, step=None, stream=None):
        out = torch.full((self.n, self.h, self.d), 77.0, dtype=torch.bfloat16, device="cuda")
        gemm.tree_attn(stream, self.q, self.h, self.kv, step or self.step(), out, gate=self.gate, scale=scale)
        return out

    def want(self, scale=None):
        """(out, tolerance) f64 [n][h][d], from the cache's codes."""
        scale = self.d**-0.5 if scale is None else scale
        host, g = Host(self.kv), self.h // self.j
        out, tol = np.zeros((2, self.n, self.h, self.d))
        q = _f64(self.q)
        for b, (a, m) in enumerate(self.seqs):
            kv = host.values(self.slots[b])
            for i in range(m):
                t = self.start[b] + i
                bits = (2 << i) - 1 if self.mask is None else int(self.mask[t])
                seen = np.r_[np.arange(a), a + np.array([s for s in range(m) if bits >> s & 1], np.int64)].astype(np.int64)
                if not len(seen):
                    continue
                for head in range(self.h):
                    k, v = kv[seen, head // g, 0], kv[seen, head // g, 1]
                    s = k @ q[t, head] * scale
                    p = np.exp(s - s.max())
                    l = p.sum()
                    out[t, head] = p @ v / l
                    # scores: sums of d products in f32, then two products; of the exponent's argument (in units of log 2)
                    # one rounding; the exponential a few units in the last place
                    ds = (np.abs(k) @ np.abs(q[t, head]) * scale * (self.d + 8) * 2.0**-24).max() + np.abs(s - s.max()).max() * 2.0**-22
                    spread = p @ np.abs(v) / l
                    # a probability times its value's scale is rounded to f16: 2^-11 of it, or half of f16's smallest step
                    # relative to the largest scale in the sequence (the reference is at most twice that)
                    vs = host.scales[self.slots[b]][:, head // g, 1]
                    small = len(seen) * 2.0**-25 * 2 * np.nanmax(vs) * TOP[self.kv.fmt] / l
                    tol[t, head] = (2.0**-11 + 4 * ds + (len(seen) + 64) * 2.0**-23) * spread + small
        if self.gate is not None:
            sig = 1 / (1 + np.exp(-_f64(self.gate)))
            out, tol = out * sig, tol * sig + np.abs(out * sig) * 2.0**-20
        return out, tol + np.abs(out) * 2.0**-8 + 1e-38

    def check(self, gemm, **kw):
        got = _f64(self.run(gemm, **kw))
        out, tol = self.want(kw.get("scale"))
        assert np.isfinite(got).all()
        off = np.abs(got - out) - tol
        assert (off <= 0).all(), (off.max(), np.unravel_index(off.argmax(), off.shape), np.abs(got - out).max())


CHAINS = [[(0, 1)], [(1, 1)], [(62, 1)], [(63, 1)], [(64, 1)], [(65, 2)], [(191, 3)], [(255, 1)], [(256, 5)], [(0, 64)], [(1000, 1)],
          [(60, 9)], [(511, 2)]]


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("seqs", CHAINS, ids=str)
def test_short_lengths(gemm, fmt, seqs):
    print(f"attention {fmt!r} {seqs}", flush=True)
    Step(seqs, fmt, 6, 1, 256, 64, gate=True).check(gemm)


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,j,page", [(1, 1, 64), (4, 4, 128), (16, 4, 256), (24, 4, 64), (7, 1, 1024), (17, 1, 64), (64, 1, 64)])
def test_head_layouts(gemm, fmt, d, h, j, page):
    print(f"attention {fmt!r} {h}/{j}x{d} page {page}", flush=True)
    Step([(300, 1), (130, 3)], fmt, h, j, d, page, seed=h).check(gemm)


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("mask", ["tree", "any", "none"])
@pytest.mark.parametrize("seqs", [[(0, 5)], [(77, 13)], [(250, 64)], [(1200, 31), (0, 64), (3, 0), (64, 1)]], ids=str)
def test_trees(gemm, fmt, mask, seqs):
    """Ancestor masks, any masks (nodes that do not see themselves), and none of the step's own tokens: with nothing cached
    such a row is empty and gives zeros."""
    print(f"tree {fmt!r} {mask} {seqs}", flush=True)
    s = Step(seqs, fmt, 6, 2, 128, 64, mask=mask, gate=True)
    s.check(gemm)
    if mask == "none" and seqs[0][0] == 0:
        assert (s.run(gemm) == 0).all()


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d,h,j", [(256, 24, 4), (128, 8, 8), (64, 4, 1)])
def test_ragged_batches(gemm, fmt, d, h, j):
    """Sequences of very different lengths share workgroups; some have nothing new, some nothing cached."""
    print(f"batch {fmt!r} {h}/{j}x{d}", flush=True)
    rng = np.random.default_rng(d)
    seqs = [(int(np.exp(rng.uniform(0, 8))), int(rng.integers(0, 4))) for _ in range(20)] + [(0, 3), (0, 0), (4000, 0), (64, 3)]
    Step(seqs, fmt, h, j, d, 128, mask="tree").check(gemm)


@pytest.mark.parametrize("fmt,seqs,h,j,d", [(KvFmt.I8, [(20001, 1)], 6, 1, 256), (KvFmt.E4M3, [(9000, 5)], 12, 2, 128),
                                            (KvFmt.I8, [(5000, 64)], 6, 2, 256), (KvFmt.E4M3, [(70000, 1)], 2, 1, 64)], ids=str)
def test_long_caches_are_joined(gemm, fmt, seqs, h, j, d):
    print(f"long {fmt!r} {seqs} {h}/{j}x{d}", flush=True)
    s = Step(seqs, fmt, h, j, d, 256, mask="tree", gate=True)
    s.check(gemm)
    assert torch.equal(s.run(gemm), s.run(gemm))


def test_many_sequences(gemm):
    """As many sequences as a step takes: the plan's last places."""
    print("1024 sequences", flush=True)
    seqs = [(b % 70, b % 3) for b in range(1024)]
    Step(seqs, KvFmt.I8, 2, 1, 64, 64).check(gemm)


def test_max_new_above_what_is_there(gemm):
    s = Step([(100, 2), (50, 1)], KvFmt.I8, 4, 2, 128, 64)
    assert torch.equal(s.run(gemm, step=s.step(64)), s.run(gemm, step=s.step(40)))
    s.check(gemm, step=s.step(64))


@pytest.mark.parametrize("scale", [1.0, 1e-4, 30.0])
def test_scales(gemm, scale):
    """A flat softmax, and one so peaked that all but one probability vanish."""
    Step([(700, 3)], KvFmt.I8, 4, 2, 128, 64).check(gemm, scale=scale)


def test_far_pages(gemm):
    """Codes past 32-bit offsets: the cache's last pages, beyond 4 GiB."""
    print("far pages", flush=True)
    per_page = 4 * 2 * 256 * 1024
    pages = (5 << 30) // per_page
    kv = KvCache.new(KvFmt.I8, 4, 256, 1024, pages)
    kv.codes.view(-1)[-8 * per_page:] = 255
    del kv
    torch.cuda.empty_cache()
    s = Far([(3000, 2)], KvFmt.I8, 8, 4, 256, 1024, gate=False, first_page=pages - 5, pages=pages)
    s.check(gemm)


class Far(Step):
    """A cache too large to look at whole: the host's copy holds its last pages."""

    def want(self, scale=None):
        last = 5
        whole, pages = self.kv, self.kv.pages
        self.kv = KvCache(whole.fmt, whole.heads, whole.head_dim, whole.page, whole.codes[pages - last:], whole.scales[pages - last:])
        slots = self.slots
        self.slots = [s - (pages - last) * whole.page for s in slots]
        try:
            return super().want(scale)
        finally:
            self.kv, self.slots = whole, slots


@pytest.mark.parametrize("fmt", list(KvFmt))
def test_unseen_values_that_are_not_finite(gemm, fmt):
    """A sibling's infinite or NaN key or value, and what lies behind the sequence's end, reach only the rows that see it."""
    s = Step([(100, 4)], fmt, 4, 2, 128, 64, mask="tree")
    s.mask[:] = [1, 2, 5, 9]  # nodes 1, 2, 3: a root, and children of node 0
    clean = s.run(gemm)
    s.k[101], s.v[102, 0, 3], s.v[103, 1, 5] = float("nan"), float("inf"), float("nan")
    kv_write(None, s.kv, s.k, s.v, s.every, 104)
    out = s.run(gemm)
    assert torch.equal(out[0], clean[0])
    assert out[1].isnan().all()  # node 1 sees its own key
    assert out[2, :2].isnan().all() and torch.equal(out[2, 2:], clean[2, 2:])
    assert out[3, 2:].isnan().all() and torch.equal(out[3, :2], clean[3, :2])


def test_queries_that_are_not_finite_or_extreme(gemm):
    s = Step([(100, 3)], KvFmt.I8, 4, 2, 128, 64)
    clean = s.run(gemm)
    s.q[1, 2, 5] = float("inf")
    s.q[2, 0, 0] = float("nan")
    out = s.run(gemm)
    assert out[1, 2].isnan().all() and out[2, 0].isnan().all()
    keep = torch.ones((3, 4), dtype=torch.bool)
    keep[1, 2] = keep[2, 0] = False
    assert torch.equal(out[keep], clean[keep])
    s = Step([(100, 2)], KvFmt.I8, 4, 2, 128, 64)
    s.q[0, 0] *= 2.0**100  # far past f16
    s.q[0, 1] *= 2.0**-120
    s.q[1, 3] = 0.0
    s.check(gemm, scale=2.0**-104)
    s.check(gemm)


def test_pages_and_lengths_that_do_not_fit(gemm):
    """They give NaN for their own sequence and touch nothing else."""
    for change in ("page", "negative page", "length", "negative length"):
        print(change, flush=True)
        s = Step([(100, 2), (600, 3), (10, 1)], KvFmt.E4M3, 4, 2, 128, 64)
        clean = s.run(gemm)
        if change == "page":
            s.table[1, 3] = s.kv.pages
        elif change == "negative page":
            s.table[1, 9] = -1
        elif change == "length":
            s.len[1] = s.table.shape[1] * 64 - 2
        else:
            s.len[1] = -1
        out = s.run(gemm)
        assert out[2:5].isnan().all(), change
        assert torch.equal(out[:2], clean[:2]) and torch.equal(out[5:], clean[5:]), change


def test_starts_that_do_not_fit_stay_in_bounds(gemm):
    for start in ([0, 2, 1, 6], [0, 2, 5, 2**31 - 1], [-5, 2, 5, 6], [0, 70, 5, 6], [9, 9, 9, 9]):
        print(start, flush=True)
        s = Step([(100, 2), (300, 3), (10, 1)], KvFmt.I8, 4, 2, 128, 64)
        guard = torch.full((8, 4, 128), 77.0, dtype=torch.bfloat16, device="cuda")
        s.start = np.array(start, np.int64).astype(np.int32)
        gemm.tree_attn(None, s.q, 4, s.kv, s.step(), guard[1:7])
        torch.cuda.synchronize()
        assert (guard[0] == 77).all() and (guard[7] == 77).all()


def test_shared_pages(gemm):
    """Two sequences over the same prefix's pages."""
    s = Step([(128, 1), (128, 1)], KvFmt.I8, 4, 1, 128, 64)
    s.table[1, :2] = s.table[0, :2]
    s.slots[1][:128] = s.slots[0][:128]
    s.check(gemm)


def test_other_stream_and_graph(gemm):
    """On a stream of its own, and captured: replays see what the buffers then hold (lengths included)."""
    s = Step([(900, 5), (40, 2)], KvFmt.I8, 24, 4, 256, 256, mask="tree", gate=True)
    step, clean = s.step(), s.run(gemm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.zeros_like(clean)
        gemm.tree_attn(side, s.q, 24, s.kv, step, out, gate=s.gate)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, clean)
    g = Graph.capture(side, lambda: gemm.tree_attn(side, s.q, 24, s.kv, step, out, gate=s.gate))
    lens = step._held[1]
    for old in (900, 500, 70, 900):
        lens[0] = old
        want = s.run(gemm, step=step)
        out.zero_()
        torch.cuda.synchronize()
        g.launch(side)
        torch.cuda.synchronize()
        assert torch.equal(out, want), old


# ---- together -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", list(KvFmt))
def test_a_step_of_a_layer(gemm, fmt):
    """Two steps as an engine runs them: prep into the cache, attention, the accepted path moved together; the second step
    attends over what the first one left."""
    h, j, d, page = 8, 2, 128, 64
    rng = np.random.default_rng(5)
    kv = new_cache(fmt, j, d, page, 4)
    table = np.array([[2, 0, 3]], np.int32)
    slot = lambda p: table[0][np.asarray(p) // page] * page + np.asarray(p) % page  # noqa: E731
    rows = AttnRows(h, j, d, d // 2, True)
    inv_freq = (1e6 ** (-np.arange(d // 4) / (d // 4))).astype(np.float32)
    w = rng.uniform(0.5, 1.5, (2, d)).astype(np.float32)
    old = 0
    for masks, depths, path in (([1, 3, 5, 0xd], [0, 1, 1, 2], [0, 2, 3]), ([1, 3, 7], [0, 1, 2], [0, 1])):
        m = len(masks)
        x = rng.standard_normal((2, m, rows.rows)).astype(np.float32)
        q, gate = torch.empty((2, m, h, d), dtype=torch.bfloat16, device="cuda")
        pos = np.array([old + e for e in depths], np.int32)
        attn_prep(None, _dev(x), 2, m, rows, _dev(w[0]), _dev(w[1]), _dev(inv_freq), _dev(pos), q, gate, kv=kv,
                  slots=_dev(slot(old + np.arange(m)).astype(np.int32)))
        s = Step.__new__(Step)
        s.seqs, s.h, s.j, s.d, s.kv, s.n = [(old, m)], h, j, d, kv, m
        s.table, s.start, s.len = table, np.array([0, m], np.int32), np.array([old], np.int32)
        s.slots, s.mask, s.q, s.gate = [slot(np.arange(old + m))], np.array(masks, np.uint64), q, gate
        s.check(gemm)
        before = Host(kv)
        src, dst = slot(old + np.array(path)), slot(old + np.arange(len(path)))
        kv_move(None, kv, _dev(src.astype(np.int32)), _dev(dst.astype(np.int32)), _dev(np.array([0, len(path)], np.int32)), 1)
        assert np.array_equal(Host(kv).codes[dst], before.codes[src])
        old += len(path)
