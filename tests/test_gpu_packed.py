"""rope_apply, append_packed, read_packed and increment_packed against plain forms."""
import numpy as np
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import KVCache, RopeTable
from airframe_amd.prompt import rope_apply
from tests.gpu_util import Pair
from tests.packed_util import DTYPES, offsets, quant_values, rand, rope_angles, rotate

pytestmark = pytest.mark.gpu
NAMES = sorted(DTYPES)


def table_of(spec):
    """The table a RopeTable.scaled(*spec) has to hold: 64-bit angles, cos and sin rounded once."""
    a = rope_angles(*spec[:7])
    mult = spec[7] if len(spec) > 7 else 1.0
    return (a.cos() * mult).float(), (a.sin() * mult).float()


# ---- rotary positions ---------------------------------------------------------------------------

@pytest.mark.parametrize("spec", [(300, 64, 10000.0, 1.0, 0, 0.0, 0.0), (131072, 128, 500000.0, 8.0, 8192, 1.0, 4.0),
                                  (40960, 96, 1e6, 4.0, 8192, 1.0, 32.0, 1.1386), (1, 2, 10000.0, 2.0, 0, 0.0, 0.0)])
def test_scaled_table(gpu, spec):
    """Entries are within one f32 rounding of the 64-bit angle's cos and sin (2^-24 mult, plus the
    64-bit sincos and angle: 2^-33 at 131072 is the most that the angle's own rounding adds)."""
    rope = RopeTable.scaled(*spec)
    cos, sin = table_of(spec)
    # identity rows give the table itself: (1, 0) pairs rotate to (cos, sin)
    n = spec[0]
    pick = torch.unique(torch.tensor([0, 1, n // 3, n // 2, n - 2, n - 1]).clamp(0, n - 1))
    rd = spec[1]
    x = torch.zeros(len(pick), 1, -(-rd // 8) * 8)
    x[..., 0:rd:2] = 1.0
    y = rope_apply(x.cuda(), pick.int().cuda(), rope).cpu()[:, 0, :rd]
    mult = spec[7] if len(spec) > 7 else 1.0
    tol = mult * (2.0 ** -23 + 2.0 ** -33)
    assert (y[:, 0::2] - cos[pick]).abs().max() <= tol
    assert (y[:, 1::2] - sin[pick]).abs().max() <= tol


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("heads,hd,rd", [(1, 8, 8), (5, 64, 64), (3, 80, 20), (8, 96, 96), (40, 128, 32), (2, 256, 254),
                                         (7, 40, 2), (33, 128, 128)])
@pytest.mark.parametrize("rows", [1, 3, 257])
def test_rope_apply(gpu, name, layout, heads, hd, rd, rows):
    """f32: the same products and sums, each rounded once, on a table that may differ from torch's in
    its last bit (2^-23 of a pair's size at most, twice).  f16 / bf16: that rounded once more."""
    dt = DTYPES[name]
    spec = (4099, rd, 10000.0, 4.0, 1024, 1.0, 8.0)
    rope = RopeTable.scaled(*spec)
    cos, sin = table_of(spec)
    x = rand((rows, heads, hd), 1, dt)
    pos = torch.from_numpy(np.random.default_rng(2).integers(0, 4099, rows).astype(np.int32))
    want = rotate(x.double(), cos.double()[pos.long()], sin.double()[pos.long()], layout)
    got = rope_apply(x.cuda(), pos.cuda(), rope, layout=layout).cpu()
    assert got.dtype == dt and got.shape == x.shape
    size = x.double().abs().amax().item() * 2  # |a cos| + |b sin|
    tol = size * 2.0 ** -21 + want.abs() * torch.finfo(dt).eps / 2
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[..., rd:], x[..., rd:])
    y = x.cuda()
    assert rope_apply(y, pos.cuda(), rope, layout=layout, out=y) is y  # in place
    assert torch.equal(y.cpu(), got)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_apply_strided_rows(gpu, layout):
    """Rows that are part of wider ones, read and written; what lies between stays."""
    rope = RopeTable.scaled(64, 64, 10000.0)
    wide = rand((31, 12, 64), 3, torch.float16).cuda()
    keep = wide.clone()
    pos = torch.arange(31, dtype=torch.int32).cuda()
    want = rope_apply(wide[:, 2:7].contiguous(), pos, rope, layout=layout)
    out = torch.full((31, 9, 64), 7.0, dtype=torch.float16, device="cuda")
    rope_apply(wide[:, 2:7], pos, rope, layout=layout, out=out[:, 1:6])
    assert torch.equal(out[:, 1:6], want) and (out[:, 0] == 7).all() and (out[:, 6:] == 7).all()
    assert torch.equal(wide, keep)
    rope_apply(wide[:, 2:7], pos, rope, layout=layout, out=wide[:, 2:7])
    assert torch.equal(wide[:, 2:7], want) and torch.equal(wide[:, :2], keep[:, :2]) and torch.equal(wide[:, 7:], keep[:, 7:])


def test_rope_apply_positions_outside(gpu):
    """A position outside the table: NaN in the rotated dims, the rest copied, other rows as ever."""
    rope = RopeTable.scaled(10, 16, 10000.0)
    x = rand((4, 2, 32), 4).cuda()
    y = rope_apply(x, torch.tensor([-1, 9, 10, 2 ** 31 - 1], dtype=torch.int32).cuda(), rope, layout="half").cpu()
    assert y[[0, 2, 3], :, :16].isnan().all() and not y[1].isnan().any()
    assert torch.equal(y[..., 16:], x.cpu()[..., 16:])


def test_rope_apply_refusals(gpu):
    rope = RopeTable.scaled(10, 16, 10000.0)
    x, pos = torch.zeros(4, 2, 16).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
    assert rope_apply(x[:0], pos[:0], rope).shape == (0, 2, 16)
    for bad in (lambda: rope_apply(x, pos.long(), rope), lambda: rope_apply(x, pos[:3], rope),
                lambda: rope_apply(x.double(), pos, rope), lambda: rope_apply(x.cpu(), pos, rope),
                lambda: rope_apply(x[..., ::2], pos, rope), lambda: rope_apply(x, pos, rope, layout="both"),
                lambda: rope_apply(x, pos, rope, out=x.half()), lambda: rope_apply(x, pos, rope, out=x[:3])):
        with pytest.raises(ValueError):
            bad()
    flat = torch.zeros(4096).cuda()
    for bad in (lambda: rope_apply(torch.zeros(4, 2, 8).cuda(), pos, rope),            # table wider than the head
                lambda: rope_apply(torch.zeros(4, 2, 20).cuda(), pos, rope),           # head_dim no multiple of 8
                lambda: rope_apply(flat[1:129].view(4, 2, 16), pos, rope),             # not 16-byte aligned
                lambda: rope_apply(flat[:128].view(4, 2, 16), pos, rope, out=flat[64:192].view(4, 2, 16))):
        with pytest.raises(TsError):
            bad()
    for spec in ((0, 16, 1e4), (4, 15, 1e4), (4, 16, 0.0), (4, 16, 1e4, 0.0), (4, 16, 1e4, 2.0, 0, 1.0, 4.0),
                 (4, 16, float("inf")), (4, 16, 1e4, 1.0, 0, 0.0, 0.0, 0.0)):
        with pytest.raises(TsError):
            RopeTable.scaled(*spec)


# ---- the cache from packed rows, and back ---------------------------------------------------------

LENS = [[1], [33], [0, 5, 0, 64, 1], [31, 32, 2, 0, 97]]


@pytest.mark.parametrize("hd", [8, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("name", NAMES)
def test_append_packed_codes(gpu, name, lens, hd):
    """Codes and scales are the oracle's bit for bit, from any type, behind existing positions, in two
    calls; a sequence without rows keeps every byte."""
    dt, n_kv, n_seq = DTYPES[name], 3, len(lens)
    pair = Pair(n_seq, n_kv, hd, 200, 10000.0)
    starts = [0, 7, 31, 32, 40][:n_seq]
    for s, a in enumerate(starts):
        if a:
            k0, v0 = (rand((1, a, n_kv, hd), 10 * s + i).numpy() for i in (1, 2))
            one = offsets([a if i == s else 0 for i in range(n_seq)])
            pair.gpu.append_packed(0, torch.from_numpy(k0[0]).cuda(), torch.from_numpy(v0[0]).cuda(), one, pair.rope)
            _oracle_append(pair.ora, s, k0[0], v0[0])
            pair.gpu.increment_packed(one)
    assert pair.gpu.seq_lens() == starts
    off = offsets(lens, first=2)
    rows = off[-1] + 3
    k, v = rand((rows, n_kv, hd), 3, dt), rand((rows, n_kv, hd), 4, dt)
    pair.gpu.append_packed(0, k.cuda(), v.cuda(), off, pair.rope)
    for s, n in enumerate(lens):
        _oracle_append(pair.ora, s, k[off[s]:off[s + 1]].float().numpy(), v[off[s]:off[s + 1]].float().numpy())
    pair.check_codes()
    pair.gpu.increment_packed(torch.tensor(off, dtype=torch.int32))
    assert pair.gpu.seq_lens() == [a + n for a, n in zip(starts, lens)]
    # the device's lengths grew too: one more row each goes right behind
    k1, v1 = rand((n_seq, n_kv, hd), 5, dt), rand((n_seq, n_kv, hd), 6, dt)
    pair.gpu.append_packed(0, k1.cuda(), v1.cuda(), offsets([1] * n_seq), pair.rope)
    for s in range(n_seq):
        _oracle_append(pair.ora, s, k1[s:s + 1].float().numpy(), v1[s:s + 1].float().numpy())
    pair.check_codes()


def _oracle_append(ora, s, k, v):
    """Append rows of one sequence to the oracle cache: all sequences get them at their lengths, the
    others' are put back."""
    n = k.shape[0]
    if n == 0:
        return
    names = ("k_packed", "v_packed", "k_scale", "v_scale")
    kept = {x: getattr(ora, x).copy() for x in names}
    lens = ora.lens.copy()
    ora.lens[:] = lens[s]
    ora.append(np.repeat(k[None], len(lens), 0), np.repeat(v[None], len(lens), 0))
    for x in names:
        now = getattr(ora, x)
        for i in range(len(lens)):
            if i != s:
                now[i] = kept[x][i]
    ora.lens[:] = lens
    ora.lens[s] += n


@pytest.mark.parametrize("hd", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("name", NAMES)
def test_read_packed_values(gpu, name, hd):
    """K and V come back as the plain quantizer's values rounded once to the type, from any start, and
    rows around them stay."""
    dt, n_kv, lens = DTYPES[name], 2, [70, 0, 33, 1]
    kv = KVCache.new_int4(2, n_kv, hd, 128, len(lens))
    off = offsets(lens)
    k, v = rand((off[-1], n_kv, hd), 1), rand((off[-1], n_kv, hd), 2)
    kv.append_packed(1, k.cuda(), v.cuda(), off, None)
    want = [torch.from_numpy(quant_values(x.numpy())) for x in (k, v)]
    got = kv.read_packed(1, off, dtype=dt)
    for g, w in zip(got, want):
        assert g.dtype == dt and torch.equal(g.cpu(), w.to(dt))
    # a part of each, into wider rows behind a gap
    pos0, n = [40, 5, 31, 0], [30, 0, 2, 1]
    part = offsets(n, first=2)
    wide = torch.full((part[-1] + 2, 3 * n_kv, hd), 9.0, dtype=dt, device="cuda")
    kv.read_packed(1, part, pos0, out=(wide[:, :n_kv], wide[:, n_kv:2 * n_kv]))
    for s in range(4):
        for i, w in enumerate(want):
            rows = w[off[s] + pos0[s]:off[s] + pos0[s] + n[s]] if n[s] else w[:0]
            assert torch.equal(wide[part[s]:part[s + 1], i * n_kv:(i + 1) * n_kv].cpu(), rows.to(dt))
    assert (wide[:, 2 * n_kv:] == 9).all() and (wide[:2] == 9).all() and (wide[-2:] == 9).all()


def test_append_packed_specials(gpu):
    """Rows of zeros, one value, the type's largest and smallest values."""
    hd = 64
    rows = torch.zeros(6, 1, hd)
    rows[1, 0, 5] = -3.0
    rows[2] = 65504.0
    rows[3, 0, ::2] = 6e-8
    rows[4] = torch.linspace(-1, 1, hd)
    rows[5, 0, 0], rows[5, 0, 1] = 1.0, 0.5
    kv = KVCache.new_int4(1, 1, hd, 8)
    for dt in DTYPES.values():
        x = rows.to(dt)
        kv.append_packed(0, x.cuda(), x.cuda(), [0, 6], None)
        k, v = kv.read_packed(0, [0, 6])
        want = torch.from_numpy(quant_values(x.float().numpy()))
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)


@pytest.mark.parametrize("n_seq", [127, 128, 129, 300])
def test_many_sequences(gpu, n_seq):
    """Batches past one launch's table."""
    g = np.random.default_rng(n_seq)
    lens = [int(x) for x in g.integers(0, 4, n_seq)]
    off = offsets(lens)
    kv = KVCache.new_int4(1, 1, 64, 8, n_seq)
    k, v = rand((off[-1], 1, 64), 1), rand((off[-1], 1, 64), 2)
    kv.append_packed(0, k.cuda(), v.cuda(), off, None)
    kv.increment_packed(off)
    assert kv.seq_lens() == lens
    gk, gv = kv.read_packed(0, off)
    assert torch.equal(gk.cpu(), torch.from_numpy(quant_values(k.numpy())))
    assert torch.equal(gv.cpu(), torch.from_numpy(quant_values(v.numpy())))
    kv.append_packed(0, k.cuda(), v.cuda(), off, None)  # at the device's new lengths
    gk, gv = kv.read_packed(0, off, lens)
    assert torch.equal(gk.cpu(), torch.from_numpy(quant_values(k.numpy())))


def test_append_packed_equals_append_quant(gpu):
    """Equal lengths, QK norm and a compacted window: the same bytes as append_quant's."""
    n_seq, n, n_kv, hd = 3, 21, 4, 128
    rope = RopeTable(256, hd, 10000.0)
    norm = (rand((hd,), 9).abs() + 0.5).cuda()
    caches = [KVCache.new_int4(1, n_kv, hd, 128, n_seq) for _ in range(2)]
    k, v = rand((n_seq, n, n_kv, hd), 1).cuda(), rand((n_seq, n, n_kv, hd), 2).cuda()
    for c in caches:
        c.set_qk_norm(0, None, norm)
        c.append_quant(0, k, v, rope)
        c.increment(n)
        c.compact(2, 9, seq=1)
    caches[0].append_quant(0, k, v, rope)
    caches[1].append_packed(0, k.view(-1, n_kv, hd), v.view(-1, n_kv, hd), offsets([n] * n_seq), rope)
    for s in range(n_seq):
        a, b = (c.export(0, s, 0, caches[0].get_seq_len(s) + n) for c in caches)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_packed_graph(gpu):
    """append, lengths and read captured once and replayed: each replay writes behind the last."""
    lens, n_kv, hd = [3, 0, 2], 2, 64
    off = offsets(lens)
    kv, eager = (KVCache.new_int4(1, n_kv, hd, 64, 3) for _ in range(2))
    rope = RopeTable(64, hd, 10000.0)
    k, v = torch.zeros(5, n_kv, hd, device="cuda"), torch.zeros(5, n_kv, hd, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kv.append_packed(0, k, v, off, rope)
            kv.increment_packed(off)
            out = kv.read_packed(0, off, [0, 0, 0])
    torch.cuda.synchronize()
    for i in range(4):
        k.copy_(rand((5, n_kv, hd), 20 + i).cuda())
        v.copy_(rand((5, n_kv, hd), 30 + i).cuda())
        graph.replay()
        eager.append_packed(0, k, v, off, rope)
        eager.increment_packed(off)
        torch.cuda.synchronize()
        for s, n in enumerate(lens):
            a, b = (c.export(0, s, 0, n * (i + 1) + 1) for c in (kv, eager))  # (and one nobody wrote)
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(x, y) for x, y in zip(out, eager.read_packed(0, off)))


def test_packed_refusals(gpu):
    kv = KVCache.new_int4(1, 2, 64, 16, 2)
    rope = RopeTable(12, 64, 10000.0)
    k = torch.zeros(20, 2, 64).cuda()
    kv.append_packed(0, k[:0], k[:0], [0, 0, 0], rope)  # nothing to do
    kv.increment_packed([4, 4, 4])
    for bad in (lambda: kv.append_packed(0, k, k, [0, 4], rope), lambda: kv.append_packed(0, k, k.half(), [0, 1, 2], rope),
                lambda: kv.append_packed(0, k, k[:5], [0, 3, 6], rope), lambda: kv.append_packed(0, k, k, [0, 3, 21], rope),
                lambda: kv.append_packed(0, k[:, :1], k, [0, 1, 2], rope), lambda: kv.append_packed(0, k.cpu(), k, [0, 1, 2], rope),
                lambda: kv.append_packed(0, k, k, torch.tensor([0, 1, 2]), rope),
                lambda: kv.read_packed(0, [0, 4, 8], [0]), lambda: kv.read_packed(0, [0, 4, 21], out=(k, k))):
        with pytest.raises(ValueError):
            bad()
    for bad, code in ((lambda: kv.append_packed(0, k, k, [0, 3, 2], rope), -1), (lambda: kv.append_packed(0, k, k, [-1, 0, 2], rope), -1),
                      (lambda: kv.append_packed(1, k, k, [0, 1, 2], rope), -1), (lambda: kv.append_packed(0, k, k, [0, 17, 18], rope), -2),
                      (lambda: kv.append_packed(0, k, k, [0, 13, 13], rope), -1), (lambda: kv.increment_packed([0, 0, 17]), -2),
                      (lambda: kv.increment_packed([0, 1, 0]), -1), (lambda: kv.read_packed(0, [0, 4, 8], [13, 0]), -1),
                      (lambda: kv.read_packed(0, [0, 4, 8], [-1, 0]), -1)):
        with pytest.raises(TsError) as e:
            bad()
        assert e.value.code == code
    assert kv.seq_lens() == [0, 0]


def test_packed_streams(gpu):
    """On a stream of the caller's, ordered by that stream alone."""
    side = torch.cuda.Stream()
    kv = KVCache.new_int4(1, 2, 128, 64, 2)
    rope = RopeTable(64, 128, 10000.0)
    off = [0, 40, 64]
    k, v = rand((64, 2, 128), 1).cuda(), rand((64, 2, 128), 2).cuda()
    pos = torch.cat([torch.arange(40), torch.arange(24)]).int().cuda()
    torch.cuda.synchronize()
    turned = rope_apply(k, pos, rope, stream=side)
    kv.append_packed(0, turned, v, off, None, stream=side)
    got = kv.read_packed(0, off, stream=side)
    side.synchronize()
    other = KVCache.new_int4(1, 2, 128, 64, 2)
    other.append_packed(0, k, v, off, rope)
    for x, y in zip(got, other.read_packed(0, off)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_append_packed_quotients_on_half_integers(gpu, name, hd):
    """16-bit rows whose elements over the scale are half-integers, and neighbours of those, at every size, with
    NaN, infinite, zero and subnormal rows: the codes of the same rows in f32 (which divide)."""
    dt, n, n_kv = DTYPES[name], 160, 3
    g = np.random.default_rng(hd)
    m = g.integers(1, 37 if name == "bf16" else 293, (n, n_kv, 1)).astype(np.float64)
    e = g.integers(*((-120, 110) if name == "bf16" else (-10, 3)), (n, n_kv, 1))
    x = m * (2 * g.integers(0, 7, (n, n_kv, hd)) + 1) / 2 * g.choice([-1.0, 1.0], (n, n_kv, hd))
    x[..., 0] = 7 * m[..., 0]
    step = torch.from_numpy(x * 2.0 ** e).to(dt).view(torch.int16)
    step += torch.from_numpy(g.choice([0, 0, 0, 1, -1], (n, n_kv, hd))).to(torch.int16)  # neighbours in the type
    v = step.view(dt)
    v[3, 0, 5:9], v[4, 1], v[5, 2, 7], v[6, 0, 2] = float("nan"), 0.0, float("inf"), float("-inf")
    v[7] = 1e-38 if name == "bf16" else 6e-8
    k = v.flip(0).contiguous()
    caches = [KVCache.new_int4(1, n_kv, hd, 200) for _ in range(2)]
    for c, (a, b) in zip(caches, ((k, v), (k.float(), v.float()))):
        c.append_packed(0, a.cuda(), b.cuda(), [0, n], None)
        c.increment(n)
    for a, b in zip(*(c.export(0, 0, 0, n) for c in caches)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_rope_table_of_another_device(gpu):
    """A table lives on one device: calls with tensors or a cache of another refuse it."""
    x, pos = torch.zeros(2, 2, 64).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    rope, kv = RopeTable(16, 64, 1e4), KVCache.new_int4(1, 2, 64, 64)
    assert rope.device == x.device == RopeTable.scaled(16, 64, 1e4).device
    rope.device = torch.device("cuda", 1)
    q = torch.zeros(1, 1, 2, 64).cuda()
    for bad in (lambda: rope_apply(x, pos, rope), lambda: kv.append_packed(0, x, x, [0, 2], rope),
                lambda: kv.attn_shared(0, q, rope, KVCache.new_int4(1, 2, 64, 64))):
        with pytest.raises(ValueError):
            bad()


def test_read_packed_rows_apart(gpu):
    """K and V into the same rows, or into rows that run into each other, is refused; interleaved they are fine."""
    kv = KVCache.new_int4(1, 2, 64, 64)
    k, v = rand((9, 2, 64), 1).cuda(), rand((9, 2, 64), 2).cuda()
    kv.append_packed(0, k, v, [0, 9], None)
    kv.increment(9)
    want = kv.read_packed(0, [0, 9])
    wide = torch.zeros(12, 5, 64, device="cuda")
    flat = wide.view(30, 2, 64)
    for a, b in ((wide[:9, :2], wide[:9, :2]), (wide[:9, :2], wide[:9, 1:3]), (wide[:9, :2], wide[1:10, 1:3]),
                 (flat[:9], flat[8:17])):
        with pytest.raises(TsError) as e:
            kv.read_packed(0, [0, 9], out=(a, b))
        assert e.value.code == -1
    kv.read_packed(0, [0, 9], out=(wide[:9, :2], wide[:9, 2:4]))
    assert torch.equal(wide[:9, :2], want[0]) and torch.equal(wide[:9, 2:4], want[1]) and (wide[:, 4] == 0).all()
    wide.zero_()
    kv.read_packed(0, [0, 9], out=(wide[:9, 3:], wide[1:10, :2]))  # (V a row further on)
    assert torch.equal(wide[:9, 3:], want[0]) and torch.equal(wide[1:10, :2], want[1]) and (wide[:, 2] == 0).all()


def test_read_packed_leading_rows(gpu):
    """Tensors that read_packed allocates have zeros in the rows before the first offset."""
    kv = KVCache.new_int4(1, 2, 64, 64, 2)
    k, v = rand((9, 2, 64), 1).cuda(), rand((9, 2, 64), 2).cuda()
    kv.append_packed(0, k, v, [0, 5, 9], None)
    want = kv.read_packed(0, [0, 5, 9])
    for dt in DTYPES.values():
        for first in (1, 300):
            full = [torch.full((first + 9, 2, 64), 3.0, dtype=dt, device="cuda") for _ in range(4)]
            del full  # (what the allocator hands out next is not zeros)
            for got, w in zip(kv.read_packed(0, [first, first + 5, first + 9], dtype=dt), want):
                assert (got[:first] == 0).all() and torch.equal(got[first:], w.to(dt))
    got = kv.read_packed(0, [7, 7, 7])  # no rows: all of them before the first
    assert all(x.shape[0] == 7 and (x == 0).all() for x in got)


def test_read_packed_positions_of_another_shape(gpu):
    """pos0 is one position a sequence: a table of them is refused, not read as its first numbers."""
    kv = KVCache.new_int4(1, 2, 64, 64, 2)
    with pytest.raises(ValueError):
        kv.read_packed(0, [0, 1, 2], torch.zeros(2, 3, dtype=torch.int32))
