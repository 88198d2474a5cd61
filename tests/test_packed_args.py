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
    for off, n_seq, rows in (([0], None, None), ([0, 2 ** 32 + 1], None, None), ([], None, None), ([0, 1], 2, None), ([0, 1, 6], 2, 5),
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


def test_cpp_mirror_compiles():
    """include/turboshimmy.hpp's packed and shared-prefix members compile as C++17, all used."""
    import os
    import subprocess
    hpp = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "turboshimmy.hpp")
    src = f"""#include "{hpp}"
namespace t = turboshimmy;
uint64_t use(t::KVCache &kv, const t::KVCache &pre, float *p, const int32_t *off, void *ws) {{
    t::RopeTable r = t::RopeTable::scaled(8, 8, 1e4, 2.0, 4, 1.0, 4.0);
    t::rope_apply(r, TS_ROPE_HALF, TS_DTYPE_F32, p, 8, off, 1, 1, 8, p, 8);
    kv.append_packed(0, TS_DTYPE_F16, p, 8, p, 8, off, &r); kv.read_packed(0, off, off, TS_DTYPE_BF16, p, 8, p, 8);
    kv.increment_packed(off); kv.share_prefix(pre, 0);
    kv.attn_shared(pre, 0, 0, p, p, p, 8, 1, r, p, ws, 0);
    t::attn_prompt(TS_DTYPE_F32, p, 8, p, 8, p, 8, off, 1, 1, 1, 8, p, 8, ws, 0);
    return t::attn_prompt_workspace(TS_DTYPE_F32, 1, 1, 8) + kv.shared_workspace_bytes(pre, 8);
}}
"""
    r = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-x", "c++", "-", "-fsyntax-only"],
                       input=src, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_more_null_handles_are_refused():
    L = load()
    off = (ctypes.c_int32 * 2)(0, 1)
    b = ctypes.c_uint64()
    assert L.ts_attn_shared_workspace(None, None, 1, 1, ctypes.byref(b)) == INVALID
    assert L.ts_attn_shared(None, None, 0, 0, None, None, None, 1, 1, None, 0.0, None, None, 0, None) == INVALID
    assert L.ts_attn_prompt_workspace(0, 10, 2, 64, ctypes.byref(b)) == 0 and b.value == 10 * 2 * (8 * 64 + 8)
    assert L.ts_attn_prompt_workspace(1, 10, 2, 64, ctypes.byref(b)) == 0 and b.value == 0
    for bad in ((3, 10, 2, 64), (0, -1, 2, 64), (0, 10, 0, 64), (0, 10, 2, 60)):
        assert L.ts_attn_prompt_workspace(*bad, ctypes.byref(b)) == INVALID
    assert L.ts_attn_prompt_workspace(0, 10, 2, 264, ctypes.byref(b)) == -3
    # a prompt call's host checks come before any device work
    p, q = 4096, 1 << 20
    ok = dict(dtype=1, q=p, qs=64, k=q, ks=64, v=q, vs=64, off=off, n=1, h=1, kv=1, hd=64, cap=0.0, out=1 << 21, os=64, ws=None, wb=0)
    def rc(**kw):
        a = dict(ok, **kw)
        return L.ts_attn_prompt(*(a[x] for x in ("dtype", "q", "qs", "k", "ks", "v", "vs", "off", "n", "h", "kv", "hd", "cap", "out",
                                                 "os", "ws", "wb")), None)
    empty = (ctypes.c_int32 * 2)(3, 3)
    assert rc(off=empty) == 0
    for kw in (dict(dtype=5), dict(q=None), dict(q=p + 8), dict(qs=63), dict(qs=68), dict(ks=1 << 23), dict(vs=(1 << 22) + 8),
               dict(n=-1), dict(h=0), dict(h=3, kv=2), dict(hd=62), dict(cap=-1.0), dict(cap=float("nan")), dict(out=p),
               dict(out=q), dict(off=(ctypes.c_int32 * 2)(1, 0)), dict(off=(ctypes.c_int32 * 2)(-1, 0)), dict(off=None),
               dict(h=64, qs=4096, os=4096, off=(ctypes.c_int32 * 2)(0, 1 << 25))):
        assert rc(**kw) == INVALID, kw
    assert rc(hd=264, qs=264, ks=264, vs=264, os=264) == -3
    assert rc(dtype=0) == -6


def test_prompt_workspace_apart():
    """A workspace that shares memory with a row of q, k, v or the output is refused, before any device work."""
    L = load()
    off = (ctypes.c_int32 * 2)(2, 12)  # rows 2 .. 11
    need = 10 * 1 * (8 * 64 + 8)
    row, at = 64 * 4, {"q": 1 << 20, "k": 2 << 20, "v": 3 << 20, "out": 4 << 20}

    def rc(ws, out=at["out"]):
        return L.ts_attn_prompt(0, at["q"], 64, at["k"], 64, at["v"], 64, off, 1, 1, 1, 64, 0.0, out, 64, ws, need, None)
    for p in at.values():
        first, end = p + 2 * row, p + 12 * row
        for ws in (first, end - 16, first - need + 16):
            assert rc(ws) == INVALID
    assert rc(8 << 20, out=at["k"] + 3 * row) == INVALID
