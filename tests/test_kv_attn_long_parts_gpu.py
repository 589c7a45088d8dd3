"""Parts of many turns: workgroups that read more than 64 tiles of one sequence (the places of the cache's tiles are looked up 64 at a
time), in each form of the kernel, and softmaxes that grow from tile to tile or stay flat over thousands of positions."""

import numpy as np
import pytest
import torch

from qwenny_amd import KvCache, KvFmt, TreeStep, kv_write
from tests.test_kv_attn_gpu import TOP, code_places

pytestmark = pytest.mark.gpu

PAGE = 256


class Long:
    """n_seq sequences of `old` + tokens positions over the same pages, position p at page order[p // PAGE % pages]: each its own
    queries. `pages` of the cache are there, fewer than positions' pages repeat."""

    def __init__(self, fmt, d, h, tokens, n_seq, old, pages, grow=0.0, larger=0.0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed + d)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.fmt, self.d, self.h, self.tokens, self.n_seq, self.old = fmt, d, h, tokens, n_seq, old
        total = old + tokens
        self.kv = KvCache.new(fmt, 1, d, PAGE, pages)
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(pages * PAGE, device="cuda")
        self.slot = (order[at // PAGE] * PAGE + at % PAGE)  # of the positions, before they repeat
        along = at[:, None] / (pages * PAGE)
        u = torch.ones(d, device="cuda") / d**0.5
        k = rand(len(at), d) + grow * along * u
        v = rand(len(at), d) * torch.exp2(larger * along)
        kv_write(None, self.kv, k.to(torch.bfloat16), v.to(torch.bfloat16), self.slot.to(torch.int32), len(at))
        self.q = (rand(n_seq * tokens, h, d) + (2 * d**0.5 * u if grow else 0)).to(torch.bfloat16)
        held = -(-total // PAGE)
        table = order[torch.arange(held, device="cuda") % pages].to(torch.int32).repeat(n_seq, 1)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.step = TreeStep(n_seq * tokens, i32(range(0, n_seq * tokens + 1, tokens)), i32([old] * n_seq), table, tokens)
        self.count = torch.bincount(torch.arange(total, device="cuda") % (pages * PAGE), minlength=pages * PAGE).double()
        self.positions = total

    def values(self):
        """Keys and values f64 [positions before they repeat][d], and the values' scales."""
        kp, vp = code_places(self.d, PAGE)
        c = self.kv.codes[:, 0]
        out = []
        for which, places in enumerate((kp, vp)):
            codes = c[:, which][:, torch.from_numpy(places).cuda()].reshape(-1, self.d)[self.slot]
            units = codes.double() - 128 if self.fmt == KvFmt.I8 else codes.view(torch.float8_e4m3fn).double()
            scales = self.kv.scales[:, 0, which].reshape(-1)[self.slot].double()
            out.append((units * scales[:, None], scales))
        return out[0][0], out[1][0], out[1][1]

    def check(self, gemm, rows, part, scale=None):
        """`rows`: of the step, to look at. `part`: positions that one workgroup sums; their results are joined."""
        out = torch.full(self.q.shape, 77.0, dtype=torch.bfloat16, device="cuda")
        gemm.tree_attn(None, self.q, self.h, self.kv, self.step, out, scale=scale)
        assert out.isfinite().all()
        scale = self.d**-0.5 if scale is None else scale
        k, v, vs = self.values()
        worst = -np.inf
        for t in rows:
            q = self.q[t].double()  # [h][d]
            count = self.count.clone()
            behind = self.tokens - 1 - t % self.tokens  # the step's tokens that a chain's token does not see
            if behind:
                last = torch.arange(self.positions - behind, self.positions, device="cuda") % len(count)
                count[last] -= 1
            s = q @ k.t() * scale
            s = torch.where(count > 0, s, -torch.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top) * count
            total = p.sum(-1, keepdim=True)
            want, spread = p @ v / total, p @ v.abs() / total
            # scores: sums of d products in f32, two products more; the exponent's argument rounded once, to half a step of the score's
            # distance from the maximum; a probability times its scale to f16, 2^-11 of it, or half of f16's smallest step relative
            # to the largest scale (the reference is at most twice that); sums of a part, then of the parts, in f32
            ds = (q.abs() @ k.abs().t() * scale * (self.d + 8) * 2.0**-24).amax(-1) + (top - torch.where(count > 0, s, top)).amax(-1) * 2.0**-22
            parts = -(-self.positions // part)
            small = count.sum() * 2.0**-25 * 2 * vs.max() * TOP[self.fmt] / total
            tol = (2.0**-11 + 4 * ds[:, None] + (part + parts + 64) * 2.0**-23) * spread + small + want.abs() * 2.0**-8
            worst = max(worst, ((out[t].double() - want).abs() - tol).max().item())
        assert worst <= 0, worst
        again = torch.zeros_like(out)
        gemm.tree_attn(None, self.q, self.h, self.kv, self.step, again, scale=scale)
        assert torch.equal(out, again)


def _part(d, waves, rows, n_seq, positions):
    """Positions of a workgroup's part: groups of 512, shared by the workgroups that the chip holds."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    each = 1 if waves == 8 else {64: 4 if rows == 16 else 3, 128: 3 if rows == 16 else 2, 256: 2}[d]
    return n_seq * -(-positions // 512) // min(cus * each, 1024) * 512


# head dimension, query heads, tokens, sequences; rows of a chunk, waves: the forms
FORMS = [(256, 6, 5, 1, 32, 8), (256, 6, 5, 2, 32, 4), (256, 4, 1, 2, 16, 4), (128, 8, 4, 2, 32, 4), (128, 4, 1, 3, 16, 4),
         (64, 8, 8, 3, 32, 4), (64, 2, 1, 4, 16, 4)]


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d,h,tokens,n_seq,rows,waves", FORMS)
def test_every_form(gemm, fmt, d, h, tokens, n_seq, rows, waves):
    old = 1_300_000
    part = _part(d, waves, rows, n_seq, old + tokens)
    print(f"{fmt!r} {h}x{d} {n_seq} sequences of {old}+{tokens}, parts of {part}", flush=True)
    assert part > 64 * 64
    s = Long(fmt, d, h, tokens, n_seq, old, 33)
    s.check(gemm, [0, tokens - 1, n_seq * tokens - 1], part, 4 * d**-0.5)  # (so peaked that a tile more or less would be seen)


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("d,h,tokens,n_seq,rows", [(64, 2, 1, 128, 16), (256, 6, 5, 64, 32)])
@pytest.mark.parametrize("grow,larger,scale", [(40.0, 0.0, None), (-40.0, 0.0, None), (0.0, 12.0, None), (0.0, -12.0, None),
                                               (40.0, 10.0, None), (0.0, 0.0, 1e-4)])
def test_growing_and_flat_softmaxes(gemm, fmt, d, h, tokens, n_seq, rows, grow, larger, scale):
    """Scores that rise (the running maximum is followed again and again) or fall, values that grow or shrink from tile to tile
    (so does what the probabilities are rounded relative to), and a flat softmax, whose sums are the longest."""
    old = 65_000
    part = _part(d, 4, rows, n_seq, old + tokens)
    print(f"{fmt!r} {h}x{d} {n_seq} sequences of {old}+{tokens}, parts of {part}: {grow} {larger} {scale}", flush=True)
    assert part > 64 * 64
    s = Long(fmt, d, h, tokens, n_seq, old, -(-(old + tokens) // PAGE), grow, larger)
    s.check(gemm, [0, tokens - 1, n_seq * tokens // 2, n_seq * tokens - 1], part, scale)
