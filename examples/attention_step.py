"""One attention layer of a model that decodes with drafted trees: a prompt, then steps that verify a tree each.

A step is the in-projection (int4), its consumer into the cache, attention over the cache and the tree, the out-projection
(int4) with its consumer, and the move of the accepted path's slots. Weights, activations and the accepted paths are made up:
the example shows the calls and their buffers. `python examples/attention_step.py` on an MI355X."""

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from qwenny_amd import AttnRows, Gemm, KvCache, KvFmt, Mat, Quant, TreeStep, add_rmsnorm, attn_prep, kv_move  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, ROT, PAGE = 1024, 8, 2, 128, 64, 64
BF16, I32 = torch.bfloat16, torch.int32


def int4(rng, rows, cols):
    """A symmetric int4 matrix, one scale for 128 columns."""
    scales = np.full(rows * cols // 128, 0.02, np.float32)
    return Quant(4, 128, rows, cols, rng.integers(0, 2**32, (rows, cols // 8), np.uint32), scales, -8 * scales)


def dev(values, dtype=I32):
    return torch.as_tensor(np.asarray(values)).to(dtype).cuda()


class Layer:
    def __init__(self, gemm, rng, pages=8):
        self.gemm = gemm
        self.rows = AttnRows(HEADS, KV_HEADS, DIM, ROT, gated=True)
        self.qkv = Mat.stack(gemm, [int4(rng, self.rows.rows, HIDDEN)])
        self.out = Mat.stack(gemm, [int4(rng, HIDDEN, HEADS * DIM)])
        self.norms = [torch.ones(n, device="cuda") for n in (DIM, DIM, HIDDEN)]
        self.inv_freq = dev(1e6 ** (-np.arange(ROT // 2) / (ROT // 2)), torch.float32)
        self.kv = KvCache.new(KvFmt.I8, KV_HEADS, DIM, PAGE, pages)
        self.pages = rng.permutation(pages)  # of the one sequence, in its positions' order
        self.table = dev(self.pages[None])

    def slots(self, positions):
        positions = np.asarray(positions)
        return self.pages[positions // PAGE] * PAGE + positions % PAGE

    def step(self, xn, h, old, depths, masks=None):
        """Tokens xn bf16 [n][HIDDEN] after `old` cached ones, at depths `depths` of their tree (None masks: a chain);
        h f32 [n][HIDDEN], the residual, is added to. Returns the next layer's bf16 input."""
        n, stream = len(depths), torch.cuda.current_stream()
        x = torch.empty((self.qkv.split(n), n, self.qkv.rows), dtype=torch.float32, device="cuda")
        splits = self.gemm.run(stream, n, self.qkv, xn, x)
        q, gate = torch.empty((2, n, HEADS, DIM), dtype=BF16, device="cuda")
        attn_prep(stream, x, splits, n, self.rows, self.norms[0], self.norms[1], self.inv_freq, dev(old + np.asarray(depths)),
                  q, gate, kv=self.kv, slots=dev(self.slots(old + np.arange(n))))
        mid = torch.empty((n, HEADS * DIM), dtype=BF16, device="cuda")
        tree = TreeStep(n, dev([0, n]), dev([old]), self.table, n, None if masks is None else dev(masks, torch.int64))
        self.gemm.tree_attn(stream, q, HEADS, self.kv, tree, mid, gate)
        y = torch.empty((self.out.split(n), n, HIDDEN), dtype=torch.float32, device="cuda")
        splits = self.gemm.run(stream, n, self.out, mid, y)
        nxt = torch.empty((n, HIDDEN), dtype=BF16, device="cuda")
        add_rmsnorm(stream, h, y, splits, n, HIDDEN, self.norms[2], nxt)
        return nxt

    def accept(self, old, path):
        """The path's tokens (numbers within the step, ascending) stay, right after the `old` ones."""
        src, dst = self.slots(old + np.asarray(path)), self.slots(old + np.arange(len(path)))
        kv_move(torch.cuda.current_stream(), self.kv, dev(src), dev(dst), dev([0, len(path)]), 1)


def main():
    rng = np.random.default_rng(0)
    gemm = Gemm.load(0)
    layer = Layer(gemm, rng)
    tokens = lambda n: (dev(rng.standard_normal((n, HIDDEN)), BF16), torch.zeros((n, HIDDEN), device="cuda"))  # noqa: E731
    old = 0
    for part in (64, 64, 5):  # a prompt of 133 tokens, up to 64 to a step
        layer.step(*tokens(part), old, range(part))
        old += part
    # trees of the last accepted token and four drafted ones, 0 -> 1 -> 2 and 0 -> 3 -> 4: a token sees itself and its ancestors
    masks, depths = [0b1, 0b11, 0b111, 0b1001, 0b11001], [0, 1, 2, 1, 2]
    for path in ([0, 1, 2], [0, 3], [0, 3, 4]):
        out = layer.step(*tokens(5), old, depths, masks)
        layer.accept(old, path)
        old += len(path)
        assert torch.isfinite(out).all()
        print(f"accepted {path}: {old} tokens in the cache, |out| {out.float().norm().item():.3f}", flush=True)
    gemm.close()


if __name__ == "__main__":
    main()
