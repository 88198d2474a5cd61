"""The packed-batch wrappers' checks that need no GPU, and the C entry points' refusals of NULL."""
import ctypes

import pytest
import torch

from airframe_amd import load
from airframe_amd import prompt as P

INVALID = -1


def test_offsets():
    for off in ([0, 3, 5], torch.tensor([0, 3, 5], dtype=torch.int32)):
        ptr, keep, n, first, last = P._offsets(off, 2, 5)
        assert (n, first, last) == (2, 0, 5) and list((ctypes.c_int32 * 3).from_address(ptr)) == [0, 3, 5]
    for off, n_seq, rows in (([0], None, None), ([], None, None), ([0, 1], 2, None), ([0, 1, 6], 2, 5),
                             (torch.tensor([0, 1]), 1, None), (torch.tensor([[0, 1]], dtype=torch.int32), 1, None),
                             (torch.tensor([0, 9, 1, 9], dtype=torch.int32)[::2], 1, None)):
        with pytest.raises(ValueError):
            P._offsets(off, n_seq, rows)


def test_rows_and_types():
    with pytest.raises(ValueError):
        P._rows(torch.zeros(2, 3, 8), None, None, None, "x")  # not on the device
    for t, h, d, dt in ((torch.zeros(2, 8), None, None, None), (torch.zeros(2, 3, 8), 4, None, None),
                        (torch.zeros(2, 3, 8), 3, 16, None), (torch.zeros(2, 3, 8), 3, 8, torch.float16)):
        with pytest.raises(ValueError):
            P._rows(t, h, d, dt, "x")
    with pytest.raises(ValueError):
        P._dtype(torch.float64, "x")


def test_null_handles_are_refused():
    L = load()
    off = (ctypes.c_int32 * 2)(0, 1)
    h = ctypes.c_void_p()
    assert L.ts_rope_create_scaled(4, 8, 1e4, 1.0, 0, 0.0, 0.0, 1.0, None) == INVALID
    for bad in ((0, 8, 1e4, 1.0, 0, 0.0, 0.0, 1.0), (4, 7, 1e4, 1.0, 0, 0.0, 0.0, 1.0), (4, 8, -1.0, 1.0, 0, 0.0, 0.0, 1.0),
                (4, 8, 1e4, float("nan"), 0, 0.0, 0.0, 1.0), (4, 8, 1e4, 1.0, 0, 1.0, 2.0, 1.0),
                (4, 8, 1e4, 1.0, 0, 0.0, 0.0, -1.0)):
        assert L.ts_rope_create_scaled(*bad, ctypes.byref(h)) == INVALID and not h
    assert L.ts_rope_apply(None, 0, 0, None, 8, None, 1, 1, 8, None, 8, None) == INVALID
    assert L.ts_append_packed(None, 0, 0, None, 8, None, 8, off, None, None) == INVALID
    assert L.ts_read_packed(None, 0, None, off, 0, None, 8, None, 8, None) == INVALID
    assert L.ts_kv_increment_packed(None, off, None) == INVALID
