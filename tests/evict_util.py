"""Plain forms of cache eviction in 64 bits, and how far f32 arithmetic may be off them."""
from __future__ import annotations

import math

import torch

from tests.packed_util import offsets, rope_angles, rotate


def cached(kv, layer, lens):
    """(K, V) of every sequence's first lens[s] slots as the codes and scales stand for them, on the CPU: a list of
    [len, heads, hd] pairs."""
    off = offsets(lens)
    k, v = (x.cpu() for x in kv.read_packed(layer, off)) if off[-1] else (None, None)
    return [(k[a:b], v[a:b]) if b > a else None for a, b in zip(off, off[1:])]


def weigh(rows, q, lens, bases, hd, rope_dim, base, softcap=0.0, q_norm=None, eps=1e-6):
    """Attention of q [n_seq, n_tok, heads, hd] over rows (cached(), the new tokens' among them) in 64 bits:
    (out, weights of every sequence, and a bound on each).

    The bound: a score is a sum over hd of products with a relative error of 24 roundings of 2^-24 (q's norm 6,
    its rotation 3 and the table's entries 1, its split into terms of 22 bits 4, the sum and the scale's product
    the rest) of the sum of their sizes A; in the exponent's domain it is rounded 4 times at the size of the
    largest score or log sum; exp2 and the sum take 16 roundings more (the approximation of exp2 is good to 2).
    An error e of every score moves a probability by 2 e of itself.  Probabilities times V's scale are kept
    in two f16 terms: 2^-20 of the value, and half of f16's smallest step (2^-25) below the window's largest,
    times a code of 7 at most."""
    n_seq, n_tok, heads, _ = q.shape
    pos = torch.tensor([[m + b + t for t in range(n_tok)] for m, b in zip(lens, bases)])
    angles = rope_angles(int(pos.max()) + 1, rope_dim, base)
    out, out_far = (torch.zeros(n_seq, n_tok, heads, hd, dtype=torch.float64) for _ in range(2))
    weights = []
    for s, m in enumerate(lens):
        x = q[s].double()
        if q_norm is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * q_norm.double()
        x = rotate(x, angles[pos[s]].cos(), angles[pos[s]].sin(), "interleaved")
        k, v = (r.double() for r in rows[s])
        n, H = k.shape[0], k.shape[1]
        g = heads // H
        seen = torch.arange(n)[None] <= m + torch.arange(n_tok)[:, None]
        w, w_far = torch.zeros(H, n, dtype=torch.float64), torch.zeros(H, n, dtype=torch.float64)
        for h in range(heads):
            kh, vh = k[:, h // g], v[:, h // g]
            sc = x[:, h] @ kh.T / math.sqrt(hd)
            size = x[:, h].abs() @ kh.abs().T / math.sqrt(hd)
            if softcap > 0.0:
                sc = softcap * torch.tanh(sc / softcap)
            sc = sc.masked_fill(~seen, -math.inf)
            p = torch.softmax(sc, -1)
            top = torch.where(seen, sc.abs(), 0.0).amax(-1) + math.log(n + 1)
            e = 2.0 ** -24 * (24 * torch.where(seen, size, 0.0).amax(-1) + 4 * 1.45 * top + 16)[:, None]
            o = p @ vh
            out[s, :, h] = o
            far = 2 * e * (p @ vh.abs()) + 2.0 ** -20 * (p @ vh.abs())
            largest = p.amax(-1, keepdim=True)
            out_far[s, :, h] = far + 2.0 ** -25 * 7 * n * largest
            w[h // g] += p.sum(0)
            w_far[h // g] += (2 * e * p).sum(0) + 2.0 ** -24 * n_tok * g * p.sum(0)
        weights.append((w, w_far))
    return out, out_far, weights


def chosen(w, lens, keep, n_sink, n_recent):
    """select_slots by sorting: w [layers, seq, heads, max_seq] on the CPU."""
    L, S, H, _ = w.shape
    out = torch.full((L, S, H, keep), -1, dtype=torch.int32)
    for s, n in enumerate(lens):
        if n <= keep:
            out[:, s, :, :n] = torch.arange(n, dtype=torch.int32)
            continue
        for i in range(L):
            for h in range(H):
                mid = range(n_sink, n - n_recent)
                key = {p: float(w[i, s, h, p]) for p in mid}
                order = sorted(mid, key=lambda p: (0 if math.isnan(key[p]) else 1, -key[p] if not math.isnan(key[p]) else 0, p))
                some = order[:keep - n_sink - n_recent]
                out[i, s, h] = torch.tensor(sorted([*range(n_sink), *some, *range(n - n_recent, n)]), dtype=torch.int32)
    return out
