"""The example of a layer's steps runs, and what it leaves in the cache is what its tokens were."""

import importlib.util
import os

import numpy as np
import pytest
import torch

from qwenny_amd import Gemm, kv_read

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "attention_step.py")


def _example():
    spec = importlib.util.spec_from_file_location("attention_step", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_runs(capfd):
    _example().main()
    lines = capfd.readouterr().out.splitlines()
    assert [x.split(":")[1].split()[0] for x in lines if x.startswith("accepted")] == ["136", "138", "141"]


def test_a_tree_s_path_is_its_chain():
    """A path of a tree gives, row by row, what the same tokens give as a chain: the rows are computed alike but for the
    order of their sums (f32, and probabilities in f16: under 2^-9 of the values, outputs in bf16: 2^-8; the norm's mean
    keeps them relative). The cache's slots of the path are the chain's, bit for bit."""
    m = _example()
    gemm = Gemm.load(0)
    masks, depths, path = [0b1, 0b11, 0b111, 0b1001, 0b11001], [0, 1, 2, 1, 2], [0, 3, 4]
    x = torch.randn((21, m.HIDDEN), generator=torch.Generator().manual_seed(1)).to(m.BF16).cuda()
    out, cached = [], []
    for tree in (True, False):
        layer = m.Layer(gemm, np.random.default_rng(3))
        zeros = lambda n: torch.zeros((n, m.HIDDEN), device="cuda")  # noqa: E731
        layer.step(x[:16].contiguous(), zeros(16), 0, range(16))
        # five tokens either way, so that the products are made in the same partials: the chain has two more at its end
        if tree:
            y = layer.step(x[16:].contiguous(), zeros(5), 16, depths, masks)[path]
            layer.accept(16, path)
        else:
            y = layer.step(x[16:][path + [1, 2]].contiguous(), zeros(5), 16, range(5))[:3]
        kv = torch.empty((2, 19, m.KV_HEADS, m.DIM), dtype=m.BF16, device="cuda")
        kv_read(None, layer.kv, m.dev(layer.slots(np.arange(19))), 19, kv[0], kv[1])
        out.append(y.float().cpu())
        cached.append(kv.float().cpu())
    assert torch.equal(cached[0], cached[1])
    rms = out[1].square().mean(-1, keepdim=True).sqrt()
    # the attention's outputs differ by two roundings to bf16 and the probabilities', the out-projection's sums average them,
    # and the result is rounded to bf16 again, twice
    assert ((out[0] - out[1]).abs() <= 2 * 2**-8 * out[1].abs() + 6 * 2**-8 * rms).all()
    gemm.close()
