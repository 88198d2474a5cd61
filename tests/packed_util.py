"""Helpers of the packed-batch tests: ragged batches and their plain forms in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def offsets(lens, first=0):
    return [first + sum(lens[:i]) for i in range(len(lens) + 1)]


def rand(shape, seed, dtype=torch.float32, scale=1.0):
    g = np.random.default_rng(seed)
    return torch.from_numpy(g.standard_normal(shape, dtype=np.float32) * np.float32(scale)).to(dtype)


def rope_angles(n_pos, rope_dim, base, factor=1.0, l_train=0, alpha=0.0, beta=0.0):
    """[n_pos, rope_dim / 2] angles in 64 bits, by the formula of ts_rope_create_scaled."""
    theta = base ** (-2.0 * torch.arange(rope_dim // 2, dtype=torch.float64) / rope_dim)
    if beta > alpha:
        ramp = ((l_train * theta / (2 * math.pi) - alpha) / (beta - alpha)).clamp(0, 1)
        theta = theta * ((1 - ramp) / factor + ramp)
    else:
        theta = theta / factor
    return torch.arange(n_pos, dtype=torch.float64)[:, None] * theta


def rotate(x, cos, sin, layout):
    """x [rows, heads, hd] and cos, sin [rows, pairs] of one type; that type throughout."""
    rd = 2 * cos.shape[-1]
    c, s, y = cos[:, None], sin[:, None], x.clone()
    a, b = (x[..., :rd // 2], x[..., rd // 2:rd]) if layout == "half" else (x[..., 0:rd:2], x[..., 1:rd:2])
    ra, rb = a * c - b * s, a * s + b * c
    if layout == "half":
        y[..., :rd // 2], y[..., rd // 2:rd] = ra, rb
    else:
        y[..., 0:rd:2], y[..., 1:rd:2] = ra, rb
    return y


def quant_values(x):
    """Rows of f32 as the INT4 codes and scales of the reference quantizer stand for them (numpy,
    one f32 rounding per operation)."""
    x = np.asarray(x, np.float32)
    m = np.abs(x).max(-1, keepdims=True)
    scale = np.where(m == 0, np.float32(1), m / np.float32(7))
    y = x / scale
    code = np.clip(np.trunc(y) + np.where(np.abs(y - np.trunc(y)) >= 0.5, np.sign(y), 0), -7, 7).astype(np.float32)
    return code * scale


def attend(q, k, v, hidden, softcap=0.0):
    """q [r, hd], k, v [n, hd], hidden [r, n]: softmax attention in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    x = q @ k.T / math.sqrt(q.shape[-1])
    if softcap > 0:
        x = softcap * torch.tanh(x / softcap)
    return torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v


def attend_bound(q, k, v, hidden, softcap=0.0):
    """attend()'s output and two lengths per element of it, in 64 bits: sqrt(sum p^2 (v - o)^2), what
    independent errors of 1 in the scores move it by, and sqrt(sum p^2 v^2), what independent relative errors
    of 1 in the rounded weights do (their sum is taken before they are rounded)."""
    q, k, v = q.double(), k.double(), v.double()
    x = q @ k.T / math.sqrt(q.shape[-1])
    if softcap > 0:
        x = softcap * torch.tanh(x / softcap)
    p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
    o, p2 = p @ v, p * p
    by_weight = p2 @ (v * v)
    by_score = (by_weight - 2 * o * (p2 @ v) + o * o * p2.sum(-1, keepdim=True)).clamp(min=0)
    return o, by_score.sqrt(), by_weight.sqrt()


def norms(x):
    """The largest element and the largest root mean square of rows."""
    x = x.double()
    return float(x.abs().max()), float(x.square().mean(-1).max().sqrt())
