"""What the packed-prompt and shared-prefix operators are timed and compared on: rotary positions
from scaled tables, the INT4 cache written from packed rows and read back, causal attention over
packed prompts, and attention of a batch behind a prefix that all of its sequences share.

A case is a dict of plain values:
  kind      "rope"    rope_apply of one tensor of head rows, each token at a position of its own
            "cache"   append_packed of ragged new rows, then read_packed of the same rows
            "prompt"  attn_prompt over packed sequences
            "shared"  attn_shared: new tokens of every sequence over the prefix and their own keys
  dtype     "f32", "f16" or "bf16": the type of the rows that go in and come out
  n_head, n_kv, head_dim, rope_dim: the head shape; n_head counts what "rope" rotates together
  n_seq, len_lo, len_hi: sequences and how many rows each brings ("shared": own cached keys),
            spread over their logarithm from the shortest to the longest
  base, factor, l_train, alpha, beta, mult, n_pos: the rotary table
Rows of quantised values come back as the values that their codes and scales stand for.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _case(kind, dtype, n_seq, len_lo, len_hi, n_head, n_kv, head_dim, **more):
    c = dict(kind=kind, dtype=dtype, n_seq=n_seq, len_lo=len_lo, len_hi=len_hi, n_head=n_head, n_kv=n_kv,
             head_dim=head_dim, rope_dim=head_dim, layout="interleaved", base=500000.0, factor=1.0, l_train=0,
             alpha=0.0, beta=0.0, mult=1.0, n_pos=32768, start=0, prefix=0, tokens=1, softcap=0.0, fused=False)
    c.update(more)
    return c


def listed():
    return [
        # One decode step of a batch: query and key heads of 32 sequences, far along in contexts
        # of up to 128K that the table is stretched for.
        _case("rope", "f32", 32, 1, 1, 40, 8, 128, start=65531, n_pos=131072, factor=8.0, l_train=8192, alpha=1.0,
              beta=4.0, name="rope_decode_b32"),
        # The query heads of a packed batch of prompts, half layout, only part of each head.
        _case("rope", "bf16", 16, 300, 2048, 32, 8, 128, rope_dim=96, layout="half", n_pos=40960, factor=4.0,
              l_train=8192, alpha=1.0, beta=32.0, mult=0.1 * math.log(4.0) + 1.0, start=1021, name="rope_prompts_half"),
        # A few new tokens for some of many sequences, as a speculative or mixed step brings them.
        _case("cache", "f16", 48, 1, 9, 32, 8, 64, start=517, name="cache_few_rows"),
        # Ragged prompts into an empty cache, rows as the QKV projection leaves them.
        _case("cache", "f32", 16, 300, 2048, 32, 8, 128, name="cache_prompts_f32"),
        # Long prompts of a model with an odd head size, behind earlier turns.
        _case("cache", "bf16", 5, 4099, 8191, 16, 8, 80, start=1003, name="cache_prompts_hd80"),
        # One short question: the latency of a call.
        _case("prompt", "f16", 1, 127, 127, 32, 8, 64, name="prompt_short_b1"),
        # A packed batch of prompts of very different lengths, read from the fused projection's rows.
        _case("prompt", "bf16", 16, 300, 2048, 32, 8, 128, fused=True, name="prompt_packed_bf16"),
        # One long document.
        _case("prompt", "f16", 1, 8192, 8192, 32, 8, 128, name="prompt_long_f16"),
        # The same in the type of this library's own activations, 256-dim heads with softcap.
        _case("prompt", "f32", 3, 501, 2100, 16, 8, 256, softcap=50.0, name="prompt_f32_hd256"),
        # A small group of chats behind a system prompt, one token each.
        _case("shared", "f32", 4, 1, 40, 32, 8, 64, prefix=1000, name="shared_decode_b4"),
        # Saturated serving behind a long document: batch 32, 8K shared keys, short turns.
        _case("shared", "f32", 32, 60, 500, 32, 8, 128, prefix=8192, name="shared_decode_b32"),
        # The first turns of eight users behind the same document: a chunk of questions at once.
        _case("shared", "f32", 8, 1, 1, 32, 8, 128, prefix=4097, tokens=256, name="shared_chunk_b8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def draw(rng):
    """A case of the listed ranges: rows of one token to long prompts, odd sizes, every type."""
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        kind = rng.choice(["rope", "cache", "prompt", "prompt", "shared", "shared"])
        n_head, n_kv, hd = rng.choice([(32, 8, 64), (24, 8, 128), (32, 8, 128), (64, 8, 128), (16, 8, 256), (16, 8, 80),
                                       (12, 4, 96)])
        n_seq = _log_int(rng, 1, 32)
        hi = _log_int(rng, 1, 8192 if kind != "shared" else 2000)
        lo = hi if rng.random() < 0.3 else _log_int(rng, 1, hi)
        more = {}
        if kind == "rope":
            more = dict(layout=rng.choice(["interleaved", "half"]), start=_log_int(rng, 1, 60000), n_pos=131072,
                        rope_dim=rng.choice([hd, hd // 2, 16 * max(1, 3 * hd // 64)]))
            if rng.random() < 0.7:
                more.update(factor=rng.choice([2.0, 4.0, 8.0, 32.0]), l_train=8192, alpha=1.0,
                            beta=rng.choice([4.0, 32.0]))
                if rng.random() < 0.5:
                    more["mult"] = 0.1 * math.log(more["factor"]) + 1.0
        elif kind == "cache":
            more = dict(start=_log_int(rng, 1, 4000) - 1)
        elif kind == "prompt":
            more = dict(softcap=rng.choice([0.0, 0.0, 50.0]), fused=rng.random() < 0.5)
        else:
            more = dict(prefix=_log_int(rng, 1, 16000), softcap=rng.choice([0.0, 0.0, 50.0]))
            if rng.random() < 0.3:
                more["tokens"] = _log_int(rng, 2, 300)
                n_seq, hi = min(n_seq, 8), min(hi, 400)
                lo = min(lo, hi)
        c = _case(kind, "f32" if kind == "shared" else rng.choice(sorted(DTYPES)), n_seq, lo, hi, n_head, n_kv, hd, **more)
        padded = c["n_seq"] * c["n_head"] * float(c["len_hi"]) ** 2 if kind == "prompt" else 0.0
        if _cost(c) <= most[kind] and padded <= 2.2e9 and (kind != "prompt" or padded * hd <= 2.8e11):
            return c


# ---- inputs ---------------------------------------------------------------------------------

def _lens(c):
    """Rows of each sequence: from len_lo to len_hi over their logarithm, in a mixed order."""
    n, lo, hi = c["n_seq"], c["len_lo"], c["len_hi"]
    if n == 1:
        return [hi]
    at = [(5 * s + n - 1) % n if n % 5 else (3 * s + n - 1) % n if n % 3 else (7 * s + n - 1) % n for s in range(n)]
    return [int(round(lo * (hi / lo) ** (a / (n - 1)))) for a in at]


def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + 7919 * what) % (1 << 62))
    return g


def _normal(seed, what, *shape):
    return torch.randn(shape, generator=_gen(seed, what), device="cuda")


def _key_rows(seed, what, n, heads, hd):
    """Key rows with the loud channels that trained models have: 2% are 6 times as large."""
    loud = torch.rand((heads, hd), generator=_gen(seed, what + 50), device="cuda") < 0.02
    return _normal(seed, what, n, heads, hd) * torch.where(loud, 6.0, 1.0)


def _inputs(c, seed):
    """Every input of a case, from the seed alone."""
    dt, hd, lens = DTYPES[c["dtype"]], c["head_dim"], _lens(c)
    n = sum(lens)
    d = {"lens": lens}
    if c["kind"] == "rope":
        pos = torch.cat([c["start"] + 17 * s + torch.arange(m, dtype=torch.int32) for s, m in enumerate(lens)])
        d.update(x=_normal(seed, 1, n, c["n_head"], hd).to(dt), pos=pos.cuda())
    elif c["kind"] == "cache":
        d.update(k=_key_rows(seed, 1, n, c["n_kv"], hd).to(dt), v=_normal(seed, 2, n, c["n_kv"], hd).to(dt),
                 start=[c["start"] + 3 * s for s in range(c["n_seq"])])
    elif c["kind"] == "prompt":
        h, kv = c["n_head"], c["n_kv"]
        q, k, v = _normal(seed, 1, n, h, hd), _normal(seed, 2, n, kv, hd), _normal(seed, 3, n, kv, hd)
        if c["fused"]:
            rows = torch.cat([q, k, v], 1).to(dt)
            q, k, v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
        d.update(q=q.to(dt), k=k.to(dt), v=v.to(dt))
    else:
        t, most = c["tokens"], max(lens) + c["tokens"]
        d.update(q=_normal(seed, 1, c["n_seq"], t, c["n_head"], hd),
                 pk=_key_rows(seed, 2, c["prefix"], c["n_kv"], hd), pv=_normal(seed, 3, c["prefix"], c["n_kv"], hd),
                 k=_key_rows(seed, 4, c["n_seq"] * most, c["n_kv"], hd).view(c["n_seq"], most, c["n_kv"], hd),
                 v=_normal(seed, 5, c["n_seq"], most, c["n_kv"], hd))
    return d


def _angles(c):
    """[n_pos, rope_dim / 2] angles in 64 bits: the pairs whose wavelength fits the trained length
    more than beta times turn as trained, those that fit it fewer than alpha times turn slower by
    the factor, those between by a mixture."""
    i = torch.arange(c["rope_dim"] // 2, dtype=torch.float64, device="cuda")
    theta = c["base"] ** (-2.0 * i / c["rope_dim"])
    if c["beta"] > c["alpha"]:
        ramp = ((c["l_train"] * theta / (2.0 * math.pi) - c["alpha"]) / (c["beta"] - c["alpha"])).clamp(0.0, 1.0)
        theta = theta * ((1.0 - ramp) / c["factor"] + ramp)
    else:
        theta = theta / c["factor"]
    return torch.arange(c["n_pos"], dtype=torch.float64, device="cuda")[:, None] * theta


def _starts(lens):
    off = torch.zeros(len(lens) + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int32), 0)
    return off


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case, seed=seed)
    lens = s["lens"]
    s["off"] = _starts(lens)
    if case["kind"] != "prompt":
        if own:
            from airframe_amd.kv_cache import RopeTable
            s["rope"] = RopeTable.scaled(case["n_pos"], case["rope_dim"], case["base"], case["factor"], case["l_train"],
                                         case["alpha"], case["beta"], case["mult"])
        else:
            a = _angles(case)
            s["cos"], s["sin"] = (a.cos() * case["mult"]).float(), (a.sin() * case["mult"]).float()
    if case["kind"] == "cache":
        # the cache with the earlier positions already in place
        if own:
            from airframe_amd.kv_cache import KVCache
            s["kv"] = KVCache.new_int4(1, case["n_kv"], case["head_dim"], max(a + b for a, b in zip(s["start"], lens)),
                                       case["n_seq"])
            for i, a in enumerate(s["start"]):
                s["kv"].set_seq_len(a, i)
            s["pos0"] = torch.tensor(s["start"], dtype=torch.int32)
        else:
            s["pos"] = torch.cat([a + torch.arange(m) for a, m in zip(s["start"], lens)]).cuda()
    elif case["kind"] == "prompt" and not own:
        at = s["off"][:-1, None] + torch.arange(max(lens))
        s["inside"] = (torch.arange(max(lens)) < torch.tensor(lens)[:, None]).cuda()
        s["rows"] = at.clamp(max=sum(lens) - 1).cuda()
    elif case["kind"] == "shared":
        if own:
            from airframe_amd.kv_cache import KVCache
            most = s["k"].shape[1]
            s["kv"] = KVCache.new_int4(1, case["n_kv"], case["head_dim"], most, case["n_seq"])
            s["kv"].requantize_all_kv_int4(0, s["k"], s["v"], most)
            s["prefix"] = KVCache.new_int4(1, case["n_kv"], case["head_dim"], case["prefix"])
            s["prefix"].requantize_all_kv_int4(0, s["pk"][None], s["pv"][None], case["prefix"])
            s["prefix"].set_seq_len(case["prefix"])
            s["kv"].share_prefix(s["prefix"])
            for i, a in enumerate(lens):
                s["kv"].set_seq_len(a, i)
            for name in ("k", "v", "pk", "pv"):
                del s[name]
        else:
            for name in ("k", "v", "pk", "pv"):
                s[name] = _codes(s[name])  # what the caches hold: codes and one scale per row
            s["len"] = torch.tensor(lens, device="cuda")
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _rotate(x, cos, sin, layout):
    """x [..., head_dim] in 32 bits by cos and sin [..., rope_dim / 2]: pairs (2i, 2i + 1), or
    (i, i + rope_dim / 2) in the half layout; dims past rope_dim stay."""
    rd = 2 * cos.shape[-1]
    rest = x[..., rd:]
    if layout == "half":
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
    else:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
    ra, rb = a * cos - b * sin, a * sin + b * cos
    y = torch.cat([ra, rb], -1) if layout == "half" else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _codes(x):
    """Bias-free 4-bit codes and the scale of each row: max |x| / 7, codes rounded half away."""
    seven = torch.full((), 7.0, device=x.device)
    scale = x.abs().amax(-1, keepdim=True) / seven
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    y = x / scale
    whole = y.trunc()
    code = whole + torch.where((y - whole).abs() >= 0.5, y.sign(), torch.zeros_like(y))
    return code.clamp(-7, 7).to(torch.int8), scale


def _values(codes):
    return codes[0].float() * codes[1]


def _cap(x, softcap):
    return torch.tanh(x / softcap) * softcap if softcap > 0.0 else x


def _softmax(x):
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_cache(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    k = _rotate(s["k"].float(), cos, sin, "interleaved")
    return [_values(_codes(k)).to(dt), _values(_codes(s["v"].float())).to(dt)]


def _plain_prompt(s):
    c = s["case"]
    n_seq, m = s["rows"].shape
    kv, g, hd = c["n_kv"], c["n_head"] // c["n_kv"], c["head_dim"]
    q = s["q"][s["rows"]].float().view(n_seq, m, kv, g, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, g * m, hd)
    k = s["k"][s["rows"]].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][s["rows"]].float().permute(0, 2, 1, 3).contiguous()
    x = _cap(torch.matmul(q, k) / math.sqrt(hd), c["softcap"]).view(n_seq, kv, g, m, m)
    hidden = torch.ones(m, m, dtype=torch.bool, device=x.device).triu(1)
    p = _softmax(x.masked_fill(hidden, -math.inf)).view(n_seq, kv, g * m, m)
    o = torch.matmul(p, v).view(n_seq, kv, g, m, hd).permute(0, 3, 1, 2, 4).reshape(n_seq, m, kv * g, hd)
    return o[s["inside"]].to(DTYPES[c["dtype"]])


def _plain_shared(s):
    c = s["case"]
    n_seq, t, kv, hd = c["n_seq"], c["tokens"], c["n_kv"], c["head_dim"]
    g = c["n_head"] // kv
    pos = c["prefix"] + s["len"][:, None] + torch.arange(t, device="cuda")
    q = _rotate(s["q"], s["cos"][pos][:, :, None], s["sin"][pos][:, :, None], "interleaved")
    q = q.view(n_seq, t, kv, g, hd).permute(2, 0, 1, 3, 4).reshape(kv, n_seq, t * g, hd)
    pk, pv, k, v = (_values(s[name]) for name in ("pk", "pv", "k", "v"))
    over = torch.matmul(q.reshape(kv, n_seq * t * g, hd), pk.permute(1, 2, 0).contiguous()).view(kv, n_seq, t * g, -1)
    mine = torch.matmul(q.permute(1, 0, 2, 3).contiguous(), k.permute(0, 2, 3, 1).contiguous()).permute(1, 0, 2, 3)
    x = _cap(torch.cat([over, mine], -1) / math.sqrt(hd), c["softcap"])
    last = (s["len"][:, None] + torch.arange(t, device="cuda"))[:, :, None].expand(-1, -1, g).reshape(n_seq, t * g, 1)
    hidden = torch.arange(-c["prefix"], k.shape[1], device="cuda") > last
    p = _softmax(x.masked_fill(hidden, -math.inf))
    o = torch.matmul(p[..., :c["prefix"]].reshape(kv, n_seq * t * g, -1), pv.permute(1, 0, 2).contiguous())
    o = o.view(kv, n_seq, t * g, hd) + torch.matmul(p[..., c["prefix"]:].permute(1, 0, 2, 3).contiguous(),
                                                   v.permute(0, 2, 1, 3).contiguous()).permute(1, 0, 2, 3)
    return o.view(kv, n_seq, t, g, hd).permute(1, 2, 0, 3, 4).reshape(n_seq, t, kv * g, hd)


def run(s):
    c = s["case"]
    if own:
        if c["kind"] == "rope":
            from airframe_amd.prompt import rope_apply
            return rope_apply(s["x"], s["pos"], s["rope"], layout=c["layout"])
        if c["kind"] == "cache":
            s["kv"].append_packed(0, s["k"], s["v"], s["off"], s["rope"])
            return list(s["kv"].read_packed(0, s["off"], s["pos0"], dtype=s["k"].dtype))
        if c["kind"] == "prompt":
            from airframe_amd.prompt import attn_prompt
            return attn_prompt(s["q"], s["k"], s["v"], s["off"], softcap=c["softcap"])
        return s["kv"].attn_shared(0, s["q"], s["rope"], s["prefix"], softcap=c["softcap"])
    if c["kind"] == "rope":
        cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
        return _rotate(s["x"].float(), cos, sin, c["layout"]).to(s["x"].dtype)
    if c["kind"] == "cache":
        return _plain_cache(s)
    return _plain_prompt(s) if c["kind"] == "prompt" else _plain_shared(s)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    c, lens = case, _lens(case)
    n, hd, size = sum(lens), c["head_dim"], SIZE[c["dtype"]]
    row4 = hd // 2 + 4  # a cached row: codes and its scale
    if c["kind"] == "rope":
        return {"bytes": 2.0 * n * c["n_head"] * hd * size + n * (4.0 * c["rope_dim"] + 4),
                "flops": 3.0 * n * c["n_head"] * c["rope_dim"]}
    if c["kind"] == "cache":
        rows = 2.0 * n * c["n_kv"]
        return {"bytes": rows * (2 * hd * size + 2 * row4) + n * 4.0 * c["rope_dim"], "flops": rows * hd * 8.0}
    if c["kind"] == "prompt":
        pairs = sum(m * (m + 1) / 2.0 for m in lens)
        return {"bytes": 2.0 * n * (c["n_head"] + c["n_kv"]) * hd * size, "flops": 4.0 * hd * c["n_head"] * pairs}
    t = c["tokens"]
    keys = sum(m + t for m in lens) + c["prefix"]
    pairs = sum(t * (c["prefix"] + m) + t * (t + 1) / 2.0 for m in lens)
    return {"bytes": 2.0 * keys * c["n_kv"] * row4 + 2.0 * c["n_seq"] * t * c["n_head"] * hd * size,
            "flops": 4.0 * hd * c["n_head"] * pairs}


# ---- in 64 bits -----------------------------------------------------------------------------------

def _turned(x, angle, mult, layout):
    """x (64 bits) as complex numbers times mult e^(i angle)."""
    rd, y = 2 * angle.shape[-1], x.clone()
    turn = torch.polar(torch.full_like(angle, mult), angle)
    if layout == "half":
        z = torch.complex(x[..., :rd // 2], x[..., rd // 2:rd]) * turn
        y[..., :rd // 2], y[..., rd // 2:rd] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rd:2].contiguous(), x[..., 1:rd:2].contiguous()) * turn
        y[..., 0:rd:2], y[..., 1:rd:2] = z.real, z.imag
    return y


def _r32(x):
    """The quantiser is defined by its roundings to 32 bits: one after each operation."""
    return x.float().double()


def _grid(x):
    """Rows of 64-bit numbers that 32 bits hold, as their 4-bit codes and scales stand for them."""
    scale = _r32(x.abs().amax(-1, keepdim=True) / 7.0)
    scale = torch.where(scale == 0, 1.0, scale)
    y = _r32(x / scale)
    return _r32(((y.abs() + 0.5).floor() * y.sign()).clamp(-7, 7) * scale)


def _attend(q, k, v, hidden, softcap):
    """q [r, hd], k and v [n, hd], hidden [r, n], all in 64 bits."""
    x = q @ k.T / math.sqrt(q.shape[-1])
    if softcap > 0.0:
        x = softcap * torch.tanh(x / softcap)
    return torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    lens, kind = d["lens"], case["kind"]
    if kind == "rope":
        return _turned(d["x"].double(), _angles(c)[d["pos"].long()][:, None], c["mult"], c["layout"])
    if kind == "cache":
        pos = torch.cat([a + torch.arange(m) for a, m in zip(d["start"], lens)]).cuda()
        angle = _angles(c)[pos][:, None]
        cos, sin = _r32(angle.cos() * c["mult"]), _r32(angle.sin() * c["mult"])
        k, rd = d["k"].double(), c["rope_dim"]
        a, b = k[..., 0:rd:2].clone(), k[..., 1:rd:2].clone()
        k[..., 0:rd:2] = _r32(_r32(a * cos) - _r32(b * sin))
        k[..., 1:rd:2] = _r32(_r32(a * sin) + _r32(b * cos))
        return [_grid(k), _grid(d["v"].double())]
    g, hd = c["n_head"] // c["n_kv"], c["head_dim"]
    if kind == "prompt":
        out, at = torch.empty(sum(lens), c["n_head"], hd, dtype=torch.float64, device="cuda"), 0
        for m in lens:
            hidden = torch.arange(m, device="cuda")[None] > torch.arange(m, device="cuda")[:, None]
            for h in range(c["n_head"]):
                q, k, v = (d[x][at:at + m, h if x == "q" else h // g].double() for x in ("q", "k", "v"))
                out[at:at + m, h] = _attend(q, k, v, hidden, c["softcap"])
            at += m
        return out
    t, angles = c["tokens"], _angles(c)
    pk, pv, k, v = (_grid(d[name].double()) for name in ("pk", "pv", "k", "v"))
    out = torch.empty(c["n_seq"], t, c["n_head"], hd, dtype=torch.float64, device="cuda")
    for s, m in enumerate(lens):
        now = torch.arange(t, device="cuda")
        q = _turned(d["q"][s].double(), angles[c["prefix"] + m + now][:, None], c["mult"], "interleaved")
        hidden = torch.arange(c["prefix"] + m + t, device="cuda")[None] > (c["prefix"] + m + now)[:, None]
        for h in range(c["n_kv"]):
            keys = torch.cat([pk[:, h], k[s, :m + t, h]])
            values = torch.cat([pv[:, h], v[s, :m + t, h]])
            rows = q[:, h * g:(h + 1) * g].reshape(t * g, hd)
            seen = hidden[:, None].expand(t, g, -1).reshape(t * g, -1)
            out[s, :, h * g:(h + 1) * g] = _attend(rows, keys, values, seen, c["softcap"]).view(t, g, hd)
    return out
