"""What the operators of cache eviction are timed and compared on: attention over the INT4 cache that
adds up what every cached slot receives, the choice of the slots that stay, and their rows moved
together, into a cache of their own.

A case is a dict of plain values:
  kind      "weigh"   attn_weigh: `tokens` new tokens of every sequence over its cached keys
            "select"  select_slots: the slots that stay, of every layer, sequence and kv head
            "keep"    keep_slots into another cache, which is then read back with read_packed
  n_head, n_kv, head_dim: the head shape
  n_seq, len_lo, len_hi: sequences and their cached slots ("weigh": before the new tokens), spread
            over their logarithm from the shortest to the longest
  spare     slots of the cache behind the longest sequence
  fresh     "weigh": the weights start at zero (else they are added to what earlier tokens left)
  n_layers, keep, n_sink, n_recent: "select" and "keep"
  dtype     "keep": the type of the rows that are read back
Rows of quantised values come back as the values that their codes and scales stand for.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BASE = 500000.0


def _case(kind, n_seq, len_lo, len_hi, n_head, n_kv, head_dim, **more):
    c = dict(kind=kind, n_seq=n_seq, len_lo=len_lo, len_hi=len_hi, n_head=n_head, n_kv=n_kv, head_dim=head_dim, spare=0)
    c.update(dict(tokens=1, fresh=True, softcap=0.0) if kind == "weigh" else dict(n_layers=1, keep=1, n_sink=0, n_recent=0))
    if kind == "keep":
        c["dtype"] = "f16"
    c.update(more)
    return c


def listed():
    return [
        # One short chat: a decode step is as long as its launches.
        _case("weigh", 1, 511, 511, 32, 8, 64, spare=512, name="weigh_decode_b1"),
        # A batch of chats of very different lengths, one token each, on top of what earlier steps left.
        _case("weigh", 8, 1001, 16003, 32, 8, 128, spare=200, fresh=False, name="weigh_decode_b8"),
        # Saturated serving: batch 32, contexts of 4K to 8K.
        _case("weigh", 32, 4096, 8192, 32, 8, 128, spare=64, name="weigh_decode_b32"),
        # Wide heads with softcap, many query heads' worth of work on few sequences.
        _case("weigh", 4, 700, 6001, 16, 8, 256, softcap=50.0, spare=1, name="weigh_decode_hd256"),
        # The last 32 tokens of four prompts look over all of it before the cache is cut.
        _case("weigh", 4, 1003, 8003, 32, 8, 128, tokens=32, spare=61, name="weigh_window_b4"),
        # One long document and a window of 64 tokens.
        _case("weigh", 1, 32704, 32704, 24, 8, 128, tokens=64, name="weigh_window_long"),
        # A prefill chunk of four sequences, its tokens' attention added up as the prompt goes in.
        _case("weigh", 4, 1024, 1536, 32, 8, 128, tokens=512, spare=512, fresh=False, name="weigh_chunk_b4"),
        # One sequence of a model with 28 layers, cut to a quarter.
        _case("select", 1, 4351, 4351, 24, 8, 128, n_layers=28, keep=1088, n_sink=4, n_recent=64, spare=100,
              name="select_b1"),
        # A batch of eight, 36 layers, long contexts of different lengths.
        _case("select", 8, 4099, 16384, 32, 8, 128, n_layers=36, keep=2048, n_sink=4, n_recent=256, spare=16,
              name="select_b8"),
        # A light cut of short chats: an eighth goes, 64-dim heads.
        _case("keep", 4, 500, 1152, 32, 8, 64, n_layers=2, keep=1008, n_sink=4, n_recent=32, spare=128, name="keep_light"),
        # One prompt from a long cache into the small one that it is continued in.
        _case("keep", 1, 15001, 15001, 32, 8, 128, n_layers=8, keep=2003, n_sink=4, n_recent=64, dtype="bf16",
              name="keep_prompt"),
        # Eight prompts cut to a quarter.
        _case("keep", 8, 2048, 8192, 32, 8, 128, n_layers=4, keep=2048, n_sink=4, n_recent=128, name="keep_b8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 4e12, w["flops"] / 1e15)


def draw(rng):
    """A case of the listed ranges: caches of one slot to long ones, odd sizes, every head shape."""
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        kind = rng.choice(["weigh", "weigh", "weigh", "select", "keep"])
        n_head, n_kv, hd = rng.choice([(32, 8, 64), (24, 8, 128), (32, 8, 128), (64, 8, 128), (16, 8, 256), (16, 8, 80),
                                       (12, 4, 96)])
        n_seq = _log_int(rng, 1, 32)
        hi = _log_int(rng, 64 if kind == "select" else 1, 32000 if kind == "weigh" else 16384)
        lo = hi if rng.random() < 0.3 else _log_int(rng, 1, hi)
        more = dict(spare=rng.choice([0, 1, 63, 500]))
        if kind == "weigh":
            more.update(fresh=rng.random() < 0.7, softcap=rng.choice([0.0, 0.0, 50.0]))
            if rng.random() < 0.5:
                more["tokens"] = _log_int(rng, 2, 512)
        else:
            # (some slots of the longest sequence are neither protected nor kept)
            keep = _log_int(rng, 8 if kind == "select" else 1, max(1, min(3 * hi // 4, 4096)))
            sink = min(keep // 2, rng.choice([0, 1, 4]))
            more.update(n_layers=_log_int(rng, 1, 36 if kind == "select" else 8), keep=keep, n_sink=sink,
                        n_recent=min((keep - sink) // 2, rng.choice([0, 16, 100, 256])))
            if kind == "keep":
                more["dtype"] = rng.choice(sorted(DTYPES))
        c = _case(kind, n_seq, lo, hi, n_head, n_kv, hd, **more)
        # (the plain form's dense arrays: padded keys and scores)
        t = c.get("tokens", 1)
        padded = c["n_seq"] * c["n_head"] * float(t) * (c["len_hi"] + t)
        dense = c.get("n_layers", 1) * c["n_seq"] * c["n_kv"] * float(c["len_hi"] + t) * hd
        if _cost(c) <= most[kind] and padded <= 2.7e8 and dense <= 4.0e8:
            return c


# ---- inputs ---------------------------------------------------------------------------------

def _lens(c):
    """Slots of each sequence: from len_lo to len_hi over their logarithm, in a mixed order."""
    n, lo, hi = c["n_seq"], c["len_lo"], c["len_hi"]
    if n == 1:
        return [hi]
    at = [(5 * s + n - 1) % n if n % 5 else (3 * s + n - 1) % n if n % 3 else (7 * s + n - 1) % n for s in range(n)]
    return [int(round(lo * (hi / lo) ** (a / (n - 1)))) for a in at]


def _slots(c):
    """Slots of one sequence's cache."""
    return max(_lens(c)) + c.get("tokens", 0) + c["spare"]


def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + 7919 * what) % (1 << 62))
    return g


def _normal(seed, what, *shape):
    return torch.randn(shape, generator=_gen(seed, what), device="cuda")


def _uniform(seed, what, *shape):
    return torch.rand(shape, generator=_gen(seed, what), device="cuda")


def _key_rows(seed, what, *shape):
    """Key rows [..., heads, hd] with the loud channels that trained models have: 2% are 6 times as large."""
    loud = _uniform(seed, what + 50, *shape[-2:]) < 0.02
    return _normal(seed, what, *shape) * torch.where(loud, 6.0, 1.0)


def _received(seed, what, lens, *shape):
    """What slots [..., seq, head, slot] have received: heavy-tailed, a tenth nothing, and no slot behind a
    sequence's last."""
    w = torch.exp(2.0 * _normal(seed, what, *shape)) * (_uniform(seed, what + 50, *shape) > 0.1)
    at = torch.arange(shape[-1], device="cuda")
    return torch.where(at < torch.tensor(lens, device="cuda")[:, None, None], w, 0.0)


def _chosen(seed, what, c, lens, n):
    """Slots that stay, drawn: the first n_sink, the last n_recent and others, ascending, -1 behind them."""
    L, S, H, keep = c["n_layers"], c["n_seq"], c["n_kv"], c["keep"]
    at, end = torch.arange(n, device="cuda"), torch.tensor(lens, device="cuda")[:, None, None]
    r = _uniform(seed, what, L, S, H, n)
    r = torch.where((at < c["n_sink"]) | (at >= end - c["n_recent"]), 2.0, r)
    r = torch.where(at < end, r, -1.0)
    slot = r.sort(dim=-1, descending=True).indices[..., :keep]
    slot = torch.where(slot < end, slot, n).sort(dim=-1).values
    return torch.where(slot < n, slot, -1).to(torch.int32)


def _inputs(c, seed):
    """Every input of a case, from the seed alone."""
    lens = _lens(c)
    S, H, hd, n = c["n_seq"], c["n_kv"], c["head_dim"], _slots(c)
    d = {"lens": lens}
    if c["kind"] == "weigh":
        full = max(lens) + c["tokens"]
        d.update(q=2.0 * _normal(seed, 1, S, c["tokens"], c["n_head"], hd), k=_key_rows(seed, 2, S, full, H, hd),
                 v=_normal(seed, 3, S, full, H, hd))
        if not c["fresh"]:
            d["w"] = _received(seed, 4, lens, S, H, n)
    elif c["kind"] == "select":
        d["w"] = _received(seed, 1, lens, c["n_layers"], S, H, n)
    else:
        d.update(k=_key_rows(seed, 1, c["n_layers"], S, max(lens), H, hd), v=_normal(seed, 2, c["n_layers"], S, max(lens), H, hd),
                 w=_received(seed, 3, lens, c["n_layers"], S, H, n), slots=_chosen(seed, 4, c, lens, max(lens)))
    return d


def _angles(c, pos):
    """Angles [..., hd / 2] of positions, in 64 bits."""
    i = torch.arange(c["head_dim"] // 2, dtype=torch.float64, device="cuda")
    return pos.double()[..., None] * BASE ** (-2.0 * i / c["head_dim"])


def _kept(c):
    """Rows that stay of each sequence, and where its rows start in the packed ones."""
    n = [min(m, c["keep"]) for m in _lens(c)]
    off = torch.zeros(len(n) + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(torch.tensor(n, dtype=torch.int32), 0)
    return n, off


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    lens, S, H, hd, n = s["lens"], case["n_seq"], case["n_kv"], case["head_dim"], _slots(case)
    if case["kind"] == "keep":
        s["off"] = _kept(case)[1]
    if own:
        from airframe_amd.kv_cache import KVCache, RopeTable
        layers = case.get("n_layers", 1)
        s["kv"] = KVCache.new_int4(layers, H, hd, n, S)
        if case["kind"] != "select":
            k, v = (s[x] if case["kind"] == "keep" else s[x][None] for x in ("k", "v"))
            for i in range(layers):
                s["kv"].requantize_all_kv_int4(i, k[i], v[i], k.shape[2])
            del s["k"], s["v"]
        for i, m in enumerate(lens):
            s["kv"].set_seq_len(m, i)
        if case["kind"] == "weigh":
            s["rope"] = RopeTable.scaled(n, hd, BASE)
            s["sum"] = torch.zeros((S, H, n), device="cuda")
        elif case["kind"] == "keep":
            s["to"] = KVCache.new_int4(layers, H, hd, case["keep"] + 64, S)
            s["sum"] = torch.zeros((layers, S, H, case["keep"] + 64), device="cuda")
    else:
        s["len"] = torch.tensor(lens, device="cuda")
        if case["kind"] == "weigh":
            pos = s["len"][:, None] + torch.arange(case["tokens"], device="cuda")
            a = _angles(case, pos)
            s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        if case["kind"] != "select":
            for x in ("k", "v"):
                s[x] = _codes(s[x])  # what the cache holds: codes and one scale per row
        if case["kind"] == "keep":
            s["inside"] = (torch.arange(case["keep"]) < torch.tensor(_kept(case)[0])[:, None]).cuda()
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _rotate(x, cos, sin):
    """x [..., hd] in 32 bits by cos and sin [..., hd / 2], pairs (2i, 2i + 1)."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _codes(x):
    """Bias-free 4-bit codes and the scale of each row: max |x| / 7, codes rounded half away."""
    seven = torch.full((), 7.0, device=x.device)
    scale = x.abs().amax(-1, keepdim=True) / seven
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    y = x / scale
    whole = y.trunc()
    code = whole + torch.where((y - whole).abs() >= 0.5, y.sign(), torch.zeros_like(y))
    return code.clamp(-7, 7).to(torch.int8), scale


def _plain_weigh(s):
    c = s["case"]
    S, t, kv, hd = c["n_seq"], c["tokens"], c["n_kv"], c["head_dim"]
    g = c["n_head"] // kv
    k, v = (s[x][0].float() * s[x][1] for x in ("k", "v"))
    q = _rotate(s["q"], s["cos"][:, :, None], s["sin"][:, :, None])
    q = q.view(S, t, kv, g, hd).permute(0, 2, 1, 3, 4).reshape(S, kv, t * g, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(hd)
    if c["softcap"] > 0.0:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    last = (s["len"][:, None] + torch.arange(t, device="cuda"))[:, :, None].expand(-1, -1, g).reshape(S, 1, t * g, 1)
    x = x.masked_fill(torch.arange(k.shape[1], device="cuda") > last, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())
    w = torch.zeros((S, kv, _slots(c)), device="cuda") if c["fresh"] else s["w"].clone()
    w[..., :k.shape[1]] += p.sum(2)
    return [o.view(S, kv, t, g, hd).permute(0, 2, 1, 3, 4).reshape(S, t, kv * g, hd), w]


def _plain_select(s):
    c, w = s["case"], s["w"]
    n = w.shape[-1]
    at, end = torch.arange(n, device="cuda"), s["len"][:, None, None]
    x = torch.where((at < c["n_sink"]) | (at >= end - c["n_recent"]), math.inf, w)
    x = torch.where(at < end, x, -math.inf)
    slot = x.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]  # equal ones in their order
    slot = torch.where(slot < end, slot, n).sort(dim=-1).values
    return torch.where(slot < n, slot, -1).to(torch.int32)


def _plain_keep(s):
    c = s["case"]
    slot = s["slots"].long()  # [layer, seq, head, keep]
    here = slot >= 0
    at = slot.clamp(min=0)
    w = torch.zeros((*slot.shape[:3], c["keep"] + 64), device="cuda")
    w[..., :c["keep"]] = torch.where(here, s["w"].gather(-1, at), 0.0)
    out = []
    at = at.permute(0, 1, 3, 2)[..., None]  # [layer, seq, keep, head, 1]
    for x in ("k", "v"):
        code, scale = s[x]
        rows = code.gather(2, at.expand(-1, -1, -1, -1, c["head_dim"])).float() * scale.gather(2, at)
        out.append(rows[:, s["inside"]].to(DTYPES[c["dtype"]]))
    return [*out, w]


def run(s):
    c = s["case"]
    if own:
        kv = s["kv"]
        if c["kind"] == "weigh":
            if not c["fresh"]:
                s["sum"].copy_(s["w"])  # (what earlier tokens left, again for every pass)
            out = kv.attn_weigh(0, s["q"], s["rope"], s["sum"], fresh=c["fresh"], softcap=c["softcap"])
            return [out, s["sum"]]
        if c["kind"] == "select":
            return kv.select_slots(s["w"], c["keep"], c["n_sink"], c["n_recent"])
        s["to"].keep_slots(s["slots"], s["sum"], src=kv, src_weights=s["w"])
        rows = int(s["off"][-1])
        k = torch.empty((c["n_layers"], rows, c["n_kv"], c["head_dim"]), dtype=DTYPES[c["dtype"]], device="cuda")
        v = torch.empty_like(k)
        for i in range(c["n_layers"]):
            s["to"].read_packed(i, s["off"], out=(k[i], v[i]))
        return [k, v, s["sum"]]
    if c["kind"] == "weigh":
        return _plain_weigh(s)
    return _plain_select(s) if c["kind"] == "select" else _plain_keep(s)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    c, lens = case, _lens(case)
    H, hd = c["n_kv"], c["head_dim"]
    row4 = hd // 2 + 4  # a cached row: codes and its scale
    if c["kind"] == "weigh":
        t = c["tokens"]
        keys = sum(m + t for m in lens)
        pairs = sum(t * m + t * (t + 1) / 2.0 for m in lens)
        return {"bytes": keys * H * (2.0 * row4 + (4 if c["fresh"] else 8)) + 8.0 * c["n_seq"] * t * c["n_head"] * hd,
                "flops": 4.0 * hd * c["n_head"] * pairs}
    kept = sum(_kept(c)[0])
    if c["kind"] == "select":
        return {"bytes": 4.0 * c["n_layers"] * H * (sum(lens) + c["n_seq"] * c["keep"]), "flops": 1.0 * c["n_layers"] * H * sum(lens)}
    rows = 1.0 * c["n_layers"] * H * kept
    return {"bytes": rows * (2 * row4 + 4 + 4 + 4 + 2 * hd * SIZE[c["dtype"]]), "flops": rows * 2 * hd}


# ---- in 64 bits -----------------------------------------------------------------------------------

def _r32(x):
    """The quantiser is defined by its roundings to 32 bits: one after each operation."""
    return x.float().double()


def _grid(x):
    """Rows of 64-bit numbers that 32 bits hold, as their 4-bit codes and scales stand for them."""
    scale = _r32(x.abs().amax(-1, keepdim=True) / 7.0)
    scale = torch.where(scale == 0, 1.0, scale)
    y = _r32(x / scale)
    return _r32(((y.abs() + 0.5).floor() * y.sign()).clamp(-7, 7) * scale)


def exact(case, seed):
    c = case
    if c["kind"] == "select":
        return None
    d = _inputs(c, seed)
    lens, H, hd = d["lens"], c["n_kv"], c["head_dim"]
    if c["kind"] == "keep":
        L, S, keep = c["n_layers"], c["n_seq"], c["keep"]
        w = torch.zeros((L, S, H, keep + 64), dtype=torch.float64, device="cuda")
        out = {x: torch.empty((L, sum(_kept(c)[0]), H, hd), dtype=torch.float64, device="cuda") for x in ("k", "v")}
        for i in range(L):
            first = 0
            for j, m in enumerate(_kept(c)[0]):
                for h in range(H):
                    at = d["slots"][i, j, h, :m].long()
                    w[i, j, h, :m] = d["w"][i, j, h, at].double()
                    for x in ("k", "v"):
                        out[x][i, first:first + m, h] = _grid(d[x][i, j, at, h].double())
                first += m
        return [out["k"], out["v"], w]
    t, g = c["tokens"], c["n_head"] // H
    out = torch.empty((c["n_seq"], t, c["n_head"], hd), dtype=torch.float64, device="cuda")
    w = torch.zeros((c["n_seq"], H, _slots(c)), dtype=torch.float64, device="cuda") if c["fresh"] else d["w"].double()
    for s, m in enumerate(lens):
        now = m + torch.arange(t, device="cuda")
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), _angles(c, now))[:, None]
        q = torch.view_as_real(torch.view_as_complex(d["q"][s].double().reshape(t, c["n_head"], hd // 2, 2)) * turn).flatten(-2)
        hidden = (torch.arange(m + t, device="cuda")[None] > now[:, None]).repeat_interleave(g, 0)
        for h in range(H):
            k, v = _grid(d["k"][s, :m + t, h].double()), _grid(d["v"][s, :m + t, h].double())
            x = q[:, h * g:(h + 1) * g].reshape(t * g, hd) @ k.T / math.sqrt(hd)
            if c["softcap"] > 0.0:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[s, :, h * g:(h + 1) * g] = (p @ v).view(t, g, hd)
            w[s, h, :m + t] += p.sum(0)
    return [out, w]
