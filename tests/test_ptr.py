"""The addresses that a call's arguments stand for, and what finding them costs."""

import timeit

import numpy as np
import pytest
import torch

from qwenny_amd.core import _ptr, _ptrs


def test_what_may_stand_for_an_address():
    t = torch.zeros(4)
    for value, want in ((None, None), (4096, 4096), (np.int64(4096), 4096), (t, t.data_ptr()), (t[1:], t.data_ptr() + 4)):
        assert _ptr(value) == want
        assert _ptrs(value, t) == [want, t.data_ptr()]
    with pytest.raises((TypeError, ValueError)):
        _ptr("text")


def test_plain_addresses_are_found_as_fast_as_tensors_are():
    """A caller that keeps addresses pays nothing for asking them whether they are tensors."""
    t = torch.zeros(4)
    took = {name: min(timeit.repeat(lambda: call(a), number=20000, repeat=9))  # noqa: B023
            for name, call, a in (("tensor", _ptr, t), ("address", _ptr, 4096), ("tensors", lambda a: _ptrs(a, a, a), t),
                                  ("addresses", lambda a: _ptrs(a, a, a), 4096))}
    # (0.6 and 0.8 times; an exception for each address makes it 2.8 times. A busy machine moves them by half)
    assert took["address"] < 1.8 * took["tensor"] and took["addresses"] < 1.8 * took["tensors"], took
