"""Eviction's refusals that need no GPU, and its C++ mirror."""
import ctypes
import os
import subprocess

from airframe_amd import load

INVALID = -1


def test_null_handles_are_refused():
    L = load()
    b = ctypes.c_uint64()
    assert L.ts_attn_weigh_workspace(None, 8, 1, ctypes.byref(b)) == INVALID
    assert L.ts_attn_weigh(None, 0, None, None, None, 8, 1, None, 0.0, None, 1, None, None, 0, None) == INVALID
    assert L.ts_kv_select(None, None, 4, 0, 0, None, None) == INVALID
    assert L.ts_kv_keep(None, 0, None, 0, 1, None, 4, None, None, None) == INVALID


def test_cpp_mirror_compiles():
    """include/turboshimmy.hpp's eviction members compile as C++17, all used."""
    hpp = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "turboshimmy.hpp")
    src = f"""#include "{hpp}"
namespace t = turboshimmy;
size_t use(t::KVCache &kv, const t::KVCache &from, const t::RopeTable &r, float *p, int32_t *slots, void *ws) {{
    kv.attn_weigh(0, p, p, p, 8, 1, r, p, true, p, ws, kv.weigh_workspace_bytes(8));
    kv.select_slots(p, 4, 1, 1, slots); kv.keep_slots(0, from, 0, 1, slots, 4, p, p); kv.keep_slots(0, from, 0, 1, slots, 4);
    kv.evict(p, 4, 0, 0, slots);
    return kv.weights_count() + kv.slots_count(4);
}}
"""
    r = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-x", "c++", "-", "-fsyntax-only"], input=src,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
