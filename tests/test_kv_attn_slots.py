"""Slots, positions and moves of another type than int32 are refused before any launch, without a GPU."""

import pytest
import torch

from qwenny_amd import AttnRows, KvCache, KvFmt, attn_prep, core, kv_move, kv_read, kv_write

heads, d, page = 2, 64, 64


class Reached(Exception):
    pass


class Lib:
    """In the library's place: host tensors never reach it, a call that would be launched says so."""

    def __getattr__(self, name):
        def call(*args):
            raise Reached(name)

        return call


@pytest.fixture
def kv(monkeypatch):
    cache = KvCache(KvFmt.I8, heads, d, page, torch.zeros((3, heads, 2, page * d), dtype=torch.uint8), torch.zeros((3, heads, 2, page)))
    monkeypatch.setattr(core, "lib", Lib)
    return cache


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.float32])
def test_types(kv, dtype):
    x = torch.zeros((2, heads, d), dtype=torch.bfloat16)
    right = torch.tensor([0, 1], dtype=torch.int32)
    wrong = right.to(dtype)
    rows = AttnRows(2, heads, d, 16)
    part, q, freq = torch.zeros((1, 2, rows.rows)), torch.zeros((2, 2, d), dtype=torch.bfloat16), torch.ones(8)
    for name, call in (("slots", lambda: kv_write(0, kv, x, x, wrong, 2)), ("slots", lambda: kv_read(0, kv, wrong, 2, x, x)),
                       ("src", lambda: kv_move(0, kv, wrong, right, right, 1)), ("dst", lambda: kv_move(0, kv, right, wrong, right, 1)),
                       ("start", lambda: kv_move(0, kv, right, right, wrong, 1)),
                       ("pos", lambda: attn_prep(0, part, 1, 2, rows, None, None, freq, wrong, q, kv=kv, slots=right)),
                       ("slots", lambda: attn_prep(0, part, 1, 2, rows, None, None, freq, right, q, kv=kv, slots=wrong))):
        with pytest.raises(ValueError, match=f"{name}.*int32"):
            call()


def test_right_types_and_addresses_reach_the_library(kv):
    x, right = torch.zeros((2, heads, d), dtype=torch.bfloat16), torch.tensor([0, 1], dtype=torch.int32)
    for slots in (right, right.data_ptr()):
        for call in (lambda: kv_write(0, kv, x, x, slots, 2), lambda: kv_read(0, kv, slots, 2, x, x),
                     lambda: kv_move(0, kv, slots, slots, slots, 1, 2),
                     lambda: attn_prep(0, x, 1, 2, AttnRows(2, heads, d), None, None, None, None, x, k=x, v=x)):
            with pytest.raises(Reached):
                call()
