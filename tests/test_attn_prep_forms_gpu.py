"""attn_prep's forms give one result: many tokens at a time (several heads to a wave, partials ahead or not, values turned over in
LDS) and token by token, bit for bit."""

import numpy as np
import pytest
import torch

from qwenny_amd import AttnRows, KvFmt, attn_prep

from tests.test_kv_attn_gpu import Host, _dev, _prep_inputs, new_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", list(KvFmt))
@pytest.mark.parametrize("h,j,d,rot,gated,splits,n", [(6, 2, 256, 64, True, 3, 70), (8, 2, 128, 128, False, 9, 130), (4, 4, 64, 16, True, 2, 520),
                                                      (5, 1, 128, 10, True, 5, 64), (4, 1, 256, 256, False, 1, 513), (2, 1, 64, 0, False, 17, 600),
                                                      (3, 3, 256, 32, True, 4, 63), (24, 4, 256, 64, True, 12, 6)])
def test_forms_agree(fmt, h, j, d, rot, gated, splits, n):
    print(f"forms {fmt!r} {h}/{j}x{d} rot {rot} gated {gated} splits {splits} n={n}", flush=True)
    rows, x, q_w, k_w, inv_freq, pos = _prep_inputs(h, j, d, rot, gated, splits, n)
    assert isinstance(rows, AttnRows)
    x, q_w, k_w, inv_freq, pos = _dev(x), _dev(q_w), _dev(k_w), _dev(inv_freq), _dev(pos)
    out = []
    slots = np.random.default_rng(n).permutation((n // 64 + 2) * 64)[:n].astype(np.int32)
    slots_dev = _dev(slots)
    for together in (True, False):
        kv = new_cache(fmt, j, d, 64, n // 64 + 2)
        q, gate = torch.zeros((2, n, h, d), dtype=torch.bfloat16, device="cuda")
        for t in [slice(0, n)] if together else [slice(i, i + 1) for i in range(n)]:
            part = x[:, t].contiguous()
            attn_prep(None, part, splits, t.stop - t.start, rows, q_w, k_w, inv_freq, pos[t], q[t], gate[t] if gated else None, kv=kv,
                      slots=slots_dev[t])
            torch.cuda.synchronize()
        host = Host(kv)
        out.append((q.cpu(), gate.cpu(), host.codes[slots], host.scales[slots]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    assert np.array_equal(out[0][2], out[1][2]) and np.array_equal(out[0][3], out[1][3])
