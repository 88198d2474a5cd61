"""Operators over packed prompts: the rows of all sequences one after another, sequence s owning rows
tok_off[s] .. tok_off[s + 1] - 1 (include/turboshimmy.h, "packed batches").  The INT4 cache's side of
them is in kv_cache.KVCache (append_packed, read_packed, increment_packed, attn_shared).

tok_off is read on the host during the call: a list of ints, or a contiguous int32 CPU tensor (which
is passed as it is).  Tensors are [rows, heads, head_dim] of float32, float16 or bfloat16; the head
rows of a token are contiguous, the distance between tokens is free, so that a slice of the fused
projection's rows can be passed as it is.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from ._lib import (TS_DTYPE_BF16, TS_DTYPE_F16, TS_DTYPE_F32, TS_ROPE_HALF, TS_ROPE_INTERLEAVED, check, load)

_DTYPE = {torch.float32: TS_DTYPE_F32, torch.float16: TS_DTYPE_F16, torch.bfloat16: TS_DTYPE_BF16}
_LAYOUT = {"interleaved": TS_ROPE_INTERLEAVED, "half": TS_ROPE_HALF}


def _dtype(dtype: torch.dtype, what: str) -> int:
    code = _DTYPE.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {dtype}")
    return code


def _rows(t: torch.Tensor, heads: int | None, head_dim: int | None, dtype: torch.dtype | None, what: str):
    """(address, stride in elements) of [rows, heads, head_dim] with contiguous head rows."""
    shape = t.shape
    if len(shape) != 3 or (heads is not None and shape[1] != heads) or (head_dim is not None and shape[2] != head_dim):
        raise ValueError(f"{what} must be [rows, {heads or 'heads'}, {head_dim or 'head_dim'}], got {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a device tensor")
    n, h, d = shape
    stride = t.stride()
    if (stride[2] != 1 and d > 1) or (stride[1] != d and h > 1):
        raise ValueError(f"{what}: the heads of a token must be contiguous")
    return t.data_ptr(), stride[0] if n > 1 else h * d


def _offsets(off, n_seq: int | None, n_rows: int | None, what: str = "tok_off"):
    """(host address, what keeps it alive, number of sequences, first and last offset) of row offsets;
    n_rows: the most rows that they may reach."""
    if isinstance(off, torch.Tensor):
        if off.dtype != torch.int32 or off.is_cuda or off.dim() != 1 or not off.is_contiguous():
            raise ValueError(f"{what} must be a list of ints or a contiguous int32 CPU tensor")
        n, ptr = off.numel(), off.data_ptr()
    else:
        n = len(off)
        if n and not (-2 ** 31 <= min(off) and max(off) < 2 ** 31):
            raise ValueError(f"{what} must be 32-bit numbers")
        off = (ctypes.c_int32 * n)(*off)
        ptr = ctypes.addressof(off)
    if n < 2 or (n_seq is not None and n != n_seq + 1):
        raise ValueError(f"{what} must hold {'at least one sequence' if n_seq is None else n_seq} + 1 offsets, got {n}")
    first, last = ctypes.c_int32.from_address(ptr).value, ctypes.c_int32.from_address(ptr + 4 * (n - 1)).value
    if n_rows is not None and last > n_rows:
        raise ValueError(f"{what} ends at row {last} of {n_rows}")
    return ptr, off, n - 1, first, last


def _same_device(first: torch.Tensor, *others):
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"arguments on {device} and {t.device}")


@contextlib.contextmanager
def _on(device: torch.device, stream):
    """The device and stream of a call as the current ones (allocations inside belong to them)."""
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
        else:
            if stream.device != device:
                raise ValueError(f"stream of {stream.device} for tensors on {device}")
            with torch.cuda.stream(stream):
                yield stream.cuda_stream


def _plain(device: torch.device, stream) -> bool:
    """Whether a call runs where the thread is already (the usual case: no contexts to enter)."""
    return stream is None and device.index == torch._C._cuda_getDevice()


def _launch(device: torch.device, stream, call):
    """call(stream address) on the device and the stream of the call."""
    if _plain(device, stream):
        return call(torch._C._cuda_getCurrentRawStream(device.index))
    with _on(device, stream) as raw:
        return call(raw)


def rope_apply(x: torch.Tensor, positions: torch.Tensor, rope, layout: str = "interleaved",
               out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Rotary positions: the first rope.rope_dim dims of every head of x [rows, heads, head_dim]
    rotated at the row's position (positions: [rows] int32 on the device), the rest copied.
    layout: pairs (2i, 2i + 1), "interleaved" as everywhere else in this library, or (i, i +
    rope_dim / 2), "half".  out may be x (in place).  A position outside the table gives NaN."""
    if layout not in _LAYOUT:
        raise ValueError(f"layout must be one of {sorted(_LAYOUT)}, got {layout!r}")
    code = _dtype(x.dtype, "x")
    px, sx = _rows(x, None, None, None, "x")
    n, heads, hd = x.shape
    if positions.dtype != torch.int32 or positions.shape != (n,) or (n > 1 and positions.stride()[0] != 1):
        raise ValueError("positions must be [rows] int32, contiguous")
    _same_device(x, positions, out, rope)
    if out is not None:
        po, so = _rows(out, heads, hd, x.dtype, "out")
        if out.shape[0] != n:
            raise ValueError(f"out must have x's {n} rows, got {out.shape[0]}")

    def call(raw):
        o, at, stride = (_fresh(x), None, heads * hd) if out is None else (out, po, so)
        check("ts_rope_apply", load().ts_rope_apply(rope.handle, _LAYOUT[layout], code, px, sx, positions.data_ptr(), n,
                                                    heads, hd, at or o.data_ptr(), stride, raw))
        return o

    return _launch(x.device, stream, call)


def _fresh(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tok_off, softcap: float = 0.0,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal attention over a packed batch of prompts: rows tok_off[s] .. tok_off[s + 1] - 1 of q
    [rows, n_head, head_dim], k and v [rows, n_head_kv, head_dim] (rotated where the model rotates;
    f32, f16 or bf16) are sequence s.  Rows outside the offsets are left as they are (zeros in an out
    allocated here).  workspace: uint8 of attn_prompt_workspace bytes (f32 only; None: allocated)."""
    code = _dtype(q.dtype, "q")
    pq, sq = _rows(q, None, None, None, "q")
    n, heads, hd = q.shape
    pk, sk = _rows(k, None, hd, q.dtype, "k")
    kv = k.shape[1]
    pv, sv = _rows(v, kv, hd, q.dtype, "v")
    off, keep, n_seq, first, last = _offsets(tok_off, None, min(n, k.shape[0], v.shape[0]))
    _same_device(q, k, v, out, workspace)
    if out is not None:
        po, so = _rows(out, heads, hd, q.dtype, "out")
        if out.shape[0] < last:
            raise ValueError(f"out has {out.shape[0]} rows, tok_off ends at {last}")

    def call(raw):
        o, at, stride = (_fresh(q), None, heads * hd) if out is None else (out, po, so)
        if out is None:
            if first > 0:
                o[:first].zero_()
            if last < n:
                o[max(last, 0):].zero_()
        ws = workspace
        if ws is None and code == TS_DTYPE_F32:
            ws = torch.empty(attn_prompt_workspace(q.dtype, max(last - first, 0), kv, hd), dtype=torch.uint8, device=q.device)
        check("ts_attn_prompt", load().ts_attn_prompt(code, pq, sq, pk, sk, pv, sv, off, n_seq, heads, kv, hd, softcap,
                                                      at or o.data_ptr(), stride, ws.data_ptr() if ws is not None else None,
                                                      ws.numel() if ws is not None else 0, raw))
        return o

    return _launch(q.device, stream, call)


def attn_prompt_workspace(dtype: torch.dtype, n_rows: int, n_head_kv: int, head_dim: int) -> int:
    """Bytes of scratch that attn_prompt needs for n_rows rows in all."""
    b = ctypes.c_uint64()
    check("ts_attn_prompt_workspace",
          load().ts_attn_prompt_workspace(_dtype(dtype, "dtype"), n_rows, n_head_kv, head_dim, ctypes.byref(b)))
    return b.value
