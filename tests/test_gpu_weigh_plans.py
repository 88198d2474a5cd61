"""attn_weigh in the forms that long and wide batches take: the integer decode kernel with its scores, with and without
splits, and chunks of more tiles of keys than the waves hold at once."""
import math

import pytest
import torch

from airframe_amd.kv_cache import KVCache, RopeTable, decode_plan
from tests.evict_util import weigh
from tests.packed_util import offsets, rand, rope_angles, rotate

pytestmark = pytest.mark.gpu
BASE = 10000.0


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def some_of(kv, layer, ends, some):
    """(K, V) of a few sequences' slots, on the CPU."""
    lens = [n if s in some else 0 for s, n in enumerate(ends)]
    off = offsets(lens)
    k, v = (x.cpu() for x in kv.read_packed(layer, off))
    return [(k[off[s]:off[s + 1]], v[off[s]:off[s + 1]]) for s in some]


def check(kv, rope_dim, q, lens, some, out, w, before=None, softcap=0.0):
    n_tok, hd, bases = q.shape[1], q.shape[3], [0] * len(some)
    ends = [m + n_tok for m in lens]
    rows = some_of(kv, 0, ends, some)
    want, far, weights = weigh(rows, q[some], [lens[s] for s in some], bases, hd, rope_dim, BASE, softcap)
    off = (out[some].cpu().double() - want).abs()
    assert bool((off <= far).all()), f"out: {float((off / far).max()):.2f} of the bound"
    for s, (ws, ws_far) in zip(some, weights):
        got, n = w[s].cpu().double(), ends[s]
        old = 0.0 if before is None else before[s, :, :n].cpu().double()
        d, limit = (got[:, :n] - old - ws).abs(), ws_far + 2.0 ** -23 * (ws + old)
        assert bool((d <= limit).all()), f"weights of {s}: {float((d / limit).max()):.2f} of the bound"
        assert torch.equal(got[:, n:], torch.zeros_like(got[:, n:]) if before is None else before[s, :, n:].cpu().double())


def batch(lens, n_tok, heads, n_kv, hd, seed):
    cap = max(lens) + n_tok + 37
    rope = RopeTable.scaled(cap, hd, BASE)
    kv = KVCache.new_int4(1, n_kv, hd, cap, len(lens))
    off = offsets(lens)
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    kv.append_packed(0, make(off[-1], n_kv, hd), make(off[-1], n_kv, hd), off, rope)
    kv.increment_packed(off)
    k, v = (make(len(lens), n_tok, n_kv, hd) for _ in range(2))
    return kv, rope, k, v, rand((len(lens), n_tok, heads, hd), seed, scale=2.0)


STEADY, LONG, RAGGED, FOUR = ([1000 + 37 * i for i in range(32)], [2601 + 37 * i for i in range(32)],
                              [1001, 16000, 3001, 5000, 7777, 2000, 1500, 9001], [700, 6001, 3001, 1500])
TOKENS = [
    # lens, heads, n_kv, hd, whether the integer kernel splits the longest sequence
    (STEADY, 128, 8, 64, False), (STEADY, 64, 8, 64, False), (STEADY, 32, 8, 64, False), (STEADY, 128, 8, 40, False),
    (LONG, 128, 8, 128, False), (LONG, 64, 8, 128, False), (STEADY, 40, 8, 96, False), (LONG, 32, 8, 256, False), (STEADY, 64, 8, 200, False),
    (RAGGED, 128, 8, 64, True), (RAGGED, 56, 8, 64, True), (RAGGED, 32, 8, 128, True), (RAGGED, 64, 8, 96, True), (RAGGED, 104, 8, 128, True),
    (RAGGED, 64, 8, 256, True), (FOUR, 16, 8, 256, True), (FOUR, 32, 8, 64, True), (FOUR, 64, 8, 200, True),
    ([20000], 24, 8, 128, True), ([30001], 64, 8, 64, True),
]


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("lens,heads,n_kv,hd,split", TOKENS)
def test_integer_kernel(lens, heads, n_kv, hd, split, append, softcap):
    plan = decode_plan([m + 1 for m in lens], n_kv, heads, hd, cus(), append)
    assert plan["integer"] and (plan["splits"] > 1) == split
    kv, rope, k, v, q = batch(lens, 1, heads, n_kv, hd, 7 + hd)
    some = [0, len(lens) - 1] + ([lens.index(max(lens))] if split else [])
    some = sorted(set(some))
    w = torch.full((len(lens), n_kv, kv.max_seq_len), float("nan"), device="cuda")
    new = dict(k=k, v=v) if append else {}
    if not append:
        kv.append_quant(0, k, v, rope)
    out = kv.attn_weigh(0, q.cuda(), rope, w, fresh=True, softcap=softcap, **new)
    check(kv, hd, q, lens, some, out, w, softcap=softcap)
    before = torch.rand(w.shape, device="cuda")
    w = before.clone()
    again = kv.attn_weigh(0, q.cuda(), rope, w, softcap=softcap, **new)
    check(kv, hd, q, lens, some, again, w, before, softcap)
    assert torch.equal(out, again)


@pytest.mark.parametrize("lens,n_tok,heads,n_kv,hd,some", [
    ([17001], 5, 16, 8, 128, [0]),          # a few columns: more tiles of keys than a workgroup's waves
    ([9001, 9500, 1], 3, 16, 8, 64, [1, 2]),
    ([9001], 4, 16, 8, 256, [0]),
    ([1100, 1500, 1321, 1234], 130, 32, 8, 128, [1, 3]),  # many: four tiles of 128-dim keys per workgroup
    ([2100, 1500, 1900, 1234], 90, 32, 8, 256, [0, 3]),
    ([1100, 1500, 1321, 1234], 130, 64, 8, 96, [0, 1]),
])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_many_tiles_of_keys(lens, n_tok, heads, n_kv, hd, some, softcap):
    kv, rope, k, v, q = batch(lens, n_tok, heads, n_kv, hd, 5 + hd)
    kv.append_quant(0, k, v, rope)
    w = torch.full((len(lens), n_kv, kv.max_seq_len), float("nan"), device="cuda")
    out = kv.attn_weigh(0, q.cuda(), rope, w, fresh=True, softcap=softcap)
    check(kv, hd, q, lens, some, out, w, softcap=softcap)
    before = torch.rand(w.shape, device="cuda")
    w = before.clone()
    assert torch.equal(kv.attn_weigh(0, q.cuda(), rope, w, softcap=softcap), out)
    check(kv, hd, q, lens, some, out, w, before, softcap)


@pytest.mark.parametrize("softcap", [0.0, 1e6])
@pytest.mark.parametrize("n_tok", [1, 5, 200])
def test_large_keys_and_small_queries(n_tok, softcap):
    """Keys of 2^114 and queries of 2^-97: products of a code sum and a key's scale alone are past f32, scores are not."""
    n_kv, heads, hd, lens = 2, 8, 128, [90, 300]
    rope = RopeTable.scaled(600, hd, BASE)
    kv = KVCache.new_int4(1, n_kv, hd, 520, 2)
    off = offsets(lens)
    kv.append_packed(0, rand((390, n_kv, hd), 1, scale=2.0 ** 114).cuda(), rand((390, n_kv, hd), 2).cuda(), off, rope)
    kv.increment_packed(off)
    kv.append_quant(0, rand((2, n_tok, n_kv, hd), 3, scale=2.0 ** 114).cuda(), rand((2, n_tok, n_kv, hd), 4).cuda(), rope)
    q = rand((2, n_tok, heads, hd), 5, scale=2.0 ** -97)
    w = torch.zeros((2, n_kv, 520), device="cuda")
    out = kv.attn_weigh(0, q.cuda(), rope, w, fresh=True, softcap=softcap)
    check(kv, hd, q, lens, [0, 1], out, w, softcap=softcap)


def columns(rows, q, m, hd):
    """The scores of one sequence's columns in 64 bits, [kv heads, columns, slots], -inf where a slot is not seen, and the
    sizes of their sums."""
    (k, _), (n_tok, heads) = rows, q.shape[:2]
    n, H = k.shape[:2]
    angles = rope_angles(m + n_tok, hd, BASE)[m:]
    x = rotate(q.double(), angles.cos(), angles.sin(), "interleaved").view(n_tok, H, heads // H, hd)
    kd = k.double().permute(1, 2, 0)
    sc = torch.stack([(x[:, h].reshape(-1, hd) @ kd[h]) / hd ** 0.5 for h in range(H)])
    size = torch.stack([(x[:, h].abs().reshape(-1, hd) @ kd[h].abs()) / hd ** 0.5 for h in range(H)])
    seen = torch.arange(n) <= m + torch.arange(n_tok).repeat_interleave(heads // H)[:, None]
    return sc.masked_fill(~seen, -torch.inf), size


@pytest.mark.parametrize("scale", [2.0 ** 14, 2.0 ** 26, 2.0 ** 60])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_tok", [1, 5, 200])
def test_scores_past_a_steps_size(n_tok, hd, scale):
    """Scores whose f32 steps reach whole numbers: a column's probabilities stay at most 1 and, with one slot far above the
    others, are one 1, whatever window it is in."""
    n_kv, heads, lens = 2, 8, [90, 700]
    kv, rope, k, v, q = batch(lens, n_tok, heads, n_kv, hd, 11)
    q = q * scale
    kv.append_quant(0, k, v, rope)
    w = torch.zeros((2, n_kv, kv.max_seq_len), device="cuda")
    out = kv.attn_weigh(0, q.cuda(), rope, w, fresh=True).cpu().double()
    ends = [m + n_tok for m in lens]
    for s, rows in enumerate(some_of(kv, 0, ends, [0, 1])):
        sc, size = columns(rows, q[s], lens[s], hd)
        top = sc.topk(2, -1)
        # a score is within 24 roundings of the size of its sum (evict_util.weigh), and behind 2^-40 of the
        # largest a slot's part is below a rounding of what it is added to
        far = 2 * 24 * 2.0 ** -24 * size.amax(-1) + 40 * math.log(2)
        clear = top.values[..., 0] - top.values[..., 1] > far
        want = torch.zeros(n_kv, ends[s], dtype=torch.float64)
        for h in range(n_kv):
            want[h].index_add_(0, top.indices[h, :, 0][clear[h]], torch.ones(int(clear[h].sum()), dtype=torch.float64))
        got = w[s, :, :ends[s]].cpu().double()
        unclear = (~clear).sum(-1)
        if scale > 2.0 ** 20:
            assert int(unclear.max()) <= 2
        # the exponent's error: the roundings of the score, the reference and the log sum (half a step each) at the largest
        # score; probabilities of 1 lose 24 roundings more in sums
        step = 2.0 ** -24 * (3 * 1.45 * float(sc.amax()) + 24)
        most = torch.exp2(torch.tensor(step if step < 1 else 0.0, dtype=torch.float64)) - 1 + 2.0 ** -20
        # a clear column leaves every other slot up to 2^-40, an unclear one any slot up to 1
        other = sc.shape[1] * 2.0 ** -40 + (1 + most) * unclear[:, None]
        off = got - want
        low, high = bool((off >= -most * want).all()), bool((off <= most * want + other).all())
        assert low and high, (float(off.min()), float(off.max()))
        # the output of a clear column is its slot's value row: kept in two f16 terms (2^-20), a sum's 24 roundings more
        v = rows[1].double()
        for h in range(n_kv):
            o = out[s, :, h * heads // n_kv:(h + 1) * heads // n_kv].reshape(-1, hd)[clear[h]]
            assert bool(((o - v[top.indices[h, :, 0][clear[h]], h]).abs() <= 2.0 ** -18 * v[:, h].abs().max()).all())
