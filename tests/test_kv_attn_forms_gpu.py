"""The attention's forms (workgroups of four and eight waves, chunks of 16 and 32 rows, groups of four and eight tiles, results
joined by the last workgroup or by a kernel of their own) and the cache's batch operators, against plain forms in 64 bits. The
forms are chosen by what a step's tables could hold, so wide tables reach each of them with few positions. Tolerances are
those of Step.want: they count the roundings."""

import numpy as np
import pytest
import torch

from qwenny_amd import Graph, KvCache, KvFmt, TreeStep, kv_read, kv_write
from tests.test_kv_attn_gpu import E4M3, TOP, Host, Step, _bf16, _dev, _f64, new_cache

pytestmark = pytest.mark.gpu

WIDE = 1 << 14  # pages of a table: positions enough for every form that many would take


class Wide(Step):
    """Tables of WIDE pages, of which the first few are looked at."""

    def __init__(self, *args, width=WIDE, **kw):
        super().__init__(*args, **kw)
        n, have = self.table.shape
        self.table = np.concatenate([self.table, np.full((n, max(0, width - have)), -7, np.int32)], 1)


# query heads, kv heads, sequences (cached, new): rows of a kv head from 1 to 448
SHAPES = [(6, 1, [(700, 1)]), (24, 4, [(1500, 1), (0, 1), (77, 1)]), (6, 1, [(700, 3)]), (6, 1, [(700, 5), (64, 2)]),
          (8, 2, [(2100, 8), (1, 0), (300, 7)]), (7, 1, [(1030, 31)]), (7, 1, [(900, 64), (10, 3)])]


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,j,seqs", SHAPES, ids=str)
def test_forms_of_long_tables(gemm, fmt, d, h, j, seqs):
    print(f"wide {fmt!r} {h}/{j}x{d} {seqs}", flush=True)
    s = Wide(seqs, fmt, h, j, d, 64, mask="tree", gate=True, seed=len(seqs))
    s.check(gemm)
    assert torch.equal(s.run(gemm), s.run(gemm))


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d,tokens", [(64, 1), (256, 1), (128, 8), (256, 8)])
def test_more_groups_than_workgroups(gemm, fmt, d, tokens):
    """Enough sequences that a workgroup has several: groups of eight tiles, parts over the borders of sequences."""
    print(f"groups {fmt!r} {d} {tokens}", flush=True)
    rng = np.random.default_rng(d + tokens)
    seqs = [(int(rng.integers(0, 700)), int(rng.integers(0, tokens + 1))) for _ in range(150)]
    Wide(seqs, fmt, 12, 4, d, 64, mask="tree", width=256).check(gemm)


def test_many_sequences_of_trees(gemm):
    print("1024 sequences of trees", flush=True)
    seqs = [(b % 130, b % 9) for b in range(1024)]
    Wide(seqs, KvFmt.E4M3, 4, 1, 128, 64, mask="tree", width=64).check(gemm)


@pytest.mark.parametrize("mask", ["any", "none"])
@pytest.mark.parametrize("d", [128, 256])
def test_masks_in_chunks_of_32_rows(gemm, mask, d):
    s = Wide([(0, 9), (200, 40), (64, 64)], KvFmt.I8, 6, 2, d, 64, mask=mask, gate=True)
    s.check(gemm)
    if mask == "none":
        assert (s.run(gemm)[:9] == 0).all()


@pytest.mark.parametrize("d,h,tokens", [(256, 6, 1), (256, 6, 5), (128, 8, 4), (256, 7, 32)])
def test_bad_pages_in_every_form(gemm, d, h, tokens):
    """A page that the cache has not, and numbers that do not fit, give NaN for their sequence alone."""
    seqs = [(300, tokens), (900, tokens), (64, tokens)]
    s = Wide(seqs, KvFmt.I8, h, 1, d, 64)
    clean = s.run(gemm)
    mine = slice(tokens, 2 * tokens)
    for change in ("page", "length"):
        t = Wide(seqs, KvFmt.I8, h, 1, d, 64)
        if change == "page":
            t.table[1, 5] = t.kv.pages
        else:
            t.len[1] = -1
        out = t.run(gemm)
        assert out[mine].isnan().all(), change
        keep = torch.ones(3 * tokens, dtype=torch.bool)
        keep[mine] = False
        assert torch.equal(out[keep], clean[keep]), change


@pytest.mark.parametrize("d,h,tokens", [(256, 6, 5), (128, 6, 8), (256, 7, 40)])
def test_not_finite_values_in_chunks_of_32_rows(gemm, d, h, tokens):
    s = Wide([(200, tokens)], KvFmt.E4M3, h, 1, d, 64, mask="tree")
    s.mask[:] = [1 << i for i in range(tokens)]  # each sees the cached positions and itself
    clean = s.run(gemm)
    s.k[200 + 1], s.v[200 + 2] = float("nan"), float("inf")
    kv_write(None, s.kv, s.k, s.v, s.every, 200 + tokens)
    out = s.run(gemm)
    assert out[1].isnan().all() and out[2].isnan().all()
    keep = [i for i in range(tokens) if i not in (1, 2)]
    assert torch.equal(out[keep], clean[keep])
    s.q[3, 0, 1] = float("nan")
    out = s.run(gemm)
    assert out[3, 0].isnan().all() and torch.equal(out[3, 1:], clean[3, 1:])


@pytest.mark.parametrize("d,h,tokens", [(256, 6, 5), (128, 6, 8), (256, 6, 1)])
def test_replays_follow_the_lengths(gemm, d, h, tokens):
    """Both ways of joining, captured: replays at other lengths than the capture's equal eager calls."""
    s = Wide([(3000, tokens)], KvFmt.I8, h, 1, d, 64, mask="tree")
    step, side = s.step(), torch.cuda.Stream()
    out = torch.zeros((tokens, h, d), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    g = Graph.capture(side, lambda: gemm.tree_attn(side, s.q, h, s.kv, step, out))
    lens = step._held[1]
    for old in (3000, 100, 1700, 0, 3000):
        lens[0] = old
        want = s.run(gemm, step=step)
        out.zero_()
        torch.cuda.synchronize()
        g.launch(side)
        torch.cuda.synchronize()
        assert torch.equal(out, want), old


# ---- the cache's batch operators ------------------------------------------------------------------------------------


def codes_f64(x, fmt):
    """The values that x's codes stand for over the scale, and the scales, in f64 on the GPU."""
    s = (x.abs().amax(-1) / TOP[fmt]).float().double()
    u = x / s[..., None]
    if fmt == KvFmt.I8:
        return u.round().clamp(-127, 127), s
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0**-6))) - 3)
    return ((u / step).round() * step).clamp(-448, 448), s


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("heads,d,page", [(2, 256, 256), (3, 128, 64), (1, 64, 1024)])
@pytest.mark.parametrize("first,n", [(0, 64), (1, 64), (37, 200), (63, 65), (3, 129), (60, 127), (130, 64)])
def test_runs_of_slots(fmt, heads, d, page, first, n):
    """A prompt's slots, from any place in a tile: written and read back, and nothing else touched."""
    print(f"run {fmt!r} {heads}x{d} page {page} {first}+{n}", flush=True)
    kv = new_cache(fmt, heads, d, page, -(-(first + n) // page) + 1)
    before = Host(kv)
    x = torch.randn((2, n, heads, d), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(torch.bfloat16)
    slots = np.arange(first, first + n)
    kv_write(None, kv, x[0], x[1], _dev(slots.astype(np.int32)), n)
    after = Host(kv)
    units, scales = codes_f64(x.double(), fmt)
    want = units.permute(1, 2, 0, 3).cpu().numpy()
    assert np.array_equal(after.units(slots), want)
    assert np.array_equal(after.scales[slots], scales.permute(1, 2, 0).float().cpu().numpy())
    rest = np.setdiff1d(np.arange(kv.pages * page), slots)
    assert np.array_equal(after.codes[rest], before.codes[rest])
    assert np.array_equal(after.scales[rest], before.scales[rest], equal_nan=True)
    k, v = torch.full_like(x, float("nan"))
    kv_read(None, kv, _dev(slots.astype(np.int32)), n, k, v)
    exact = (want.astype(np.float32) * after.scales[slots][..., None]).astype(np.float64)
    assert np.array_equal(np.stack([_f64(k), _f64(v)], 2), _bf16(exact))


@pytest.mark.parametrize("fmt", list(KvFmt))
def test_codes_are_the_nearest(fmt):
    """Four million quotients, values next to a code's border among them: each code is the nearest, ties to even."""
    n, heads, d = 2048, 4, 256
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((2, n, heads, d), generator=g, device="cuda") * torch.exp2(torch.randint(-60, 60, (2, n, heads, 1), generator=g, device="cuda"))
    x[:, ::3] = x[:, ::3].abs().round()  # few bits: quotients on borders
    x[:, 1::3] = (torch.randint(-254, 255, (2, len(range(1, n, 3)), heads, d), generator=g, device="cuda") / 2).float()
    x[:, 1::3, :, 0] = 127.0  # scale 1: whole and half numbers
    x[:, :, :, 1] = x[:, :, :, 1].abs() + 1e-20
    x = x.to(torch.bfloat16)
    kv = KvCache.new(fmt, heads, d, 256, n // 256)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    kv_write(None, kv, x[0], x[1], slots, n)
    units, scales = codes_f64(x.double(), fmt)
    host = Host(kv)
    assert np.array_equal(host.units(slice(0, n)), units.permute(1, 2, 0, 3).cpu().numpy())
    assert np.array_equal(host.scales, scales.permute(1, 2, 0).float().cpu().numpy())


@pytest.mark.parametrize("fmt", list(KvFmt))
def test_many_slots_out_of_order_repeated_and_outside(fmt):
    kv = new_cache(fmt, 2, 128, 64, 9)
    rng = np.random.default_rng(3)
    n = 150
    slots = rng.permutation(9 * 64)[:n].astype(np.int32)
    slots[[5, 70, 149]] = [-1, 9 * 64, 2**31 - 1]
    x = torch.randn((2, n, 2, 128), device="cuda").to(torch.bfloat16)
    x[0, 20, 1, 3], x[1, 30, 0, 7] = float("inf"), float("nan")
    kv_write(None, kv, x[0], x[1], _dev(slots), n)
    host = Host(kv)
    inside = (slots >= 0) & (slots < 9 * 64)
    assert np.isnan(host.scales[slots[20], 1, 0]) and np.isnan(host.scales[slots[30], 0, 1])
    again = slots[rng.integers(0, n, 200)]  # read: slots may repeat
    k, v = torch.full((2, 200, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    kv_read(None, kv, _dev(again), 200, k, v)
    ok = (again >= 0) & (again < 9 * 64)
    at = again[ok]
    exact = (host.units(at).astype(np.float32) * host.scales[at][..., None]).astype(np.float64)
    got = np.stack([_f64(k), _f64(v)], 2)
    assert np.array_equal(got[ok], _bf16(exact), equal_nan=True)
    assert (got[~ok] == 0).all()
    rest = np.setdiff1d(np.arange(9 * 64), slots[inside])
    clean = Host(new_cache(fmt, 2, 128, 64, 9))
    assert np.array_equal(host.codes[rest], clean.codes[rest])


def test_scales_below_the_normal_numbers_stay_finite():
    for fmt in KvFmt:
        kv = new_cache(fmt, 1, 64, 64, 2)
        x = (torch.finfo(torch.float32).tiny * torch.randn((2, 70, 1, 64), device="cuda")).to(torch.bfloat16)
        slots = torch.arange(70, dtype=torch.int32, device="cuda")
        kv_write(None, kv, x[0], x[1], slots, 70)
        host = Host(kv)
        assert np.isfinite(host.units(slice(0, 70))).all() and np.isfinite(host.scales[:70]).all()
        assert len(E4M3) == 256


def test_step_holds_its_tensors():
    """A TreeStep keeps its arrays: freed ones would be read."""
    s = Step([(100, 1)], KvFmt.I8, 4, 2, 64, 64)
    step = s.step()
    assert isinstance(step, TreeStep) and all(t is None or t.is_cuda for t in step._held)
