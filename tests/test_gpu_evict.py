"""select_slots, keep_slots and evict against sorting and indexing."""
import math

import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import KVCache, RopeTable
from tests.evict_util import cached, chosen, weigh
from tests.packed_util import offsets, rand

pytestmark = pytest.mark.gpu
BASE = 10000.0


def cache(lens, n_layers, n_kv, hd, cap=None, seed=0, rope=None):
    """A cache of n_layers whose sequences hold lens[s] random slots."""
    kv = KVCache.new_int4(n_layers, n_kv, hd, cap or max(max(lens), 1), len(lens))
    off = offsets(lens)
    if off[-1]:
        for i in range(n_layers):
            kv.append_packed(i, rand((off[-1], n_kv, hd), seed + 2 * i).cuda(), rand((off[-1], n_kv, hd), seed + 2 * i + 1).cuda(), off, rope)
        kv.increment_packed(off)
    return kv


WEIGHTS = {
    "normal": lambda s: torch.exp(2 * rand(s, 1)),
    "ties": lambda s: (3 * rand(s, 2)).round(),
    "zeros": lambda s: torch.zeros(s),
    "mostly_zeros": lambda s: torch.where(rand(s, 3) > 1.5, rand(s, 4).abs(), 0.0),
    "tiny": lambda s: rand(s, 5).abs() * 2.0 ** -140,
    "mixed": lambda s: torch.where(rand(s, 6) > 1, math.inf, torch.where(rand(s, 7) > 1, math.nan, torch.where(
        rand(s, 8) > 1, -math.inf, torch.where(rand(s, 9) > 0, -0.0, 0.0)))),
    "one_step": lambda s: torch.nextafter(torch.ones(s), torch.full(s, 2.0)) - (rand(s, 10) > 0).float() * 2.0 ** -23,
    "rising": lambda s: torch.arange(math.prod(s), dtype=torch.float32).view(s),
    "far_apart": lambda s: torch.where(rand(s, 11) > 0, 1e38, 1e-38) * (1 + rand(s, 12).abs()),
}


@pytest.mark.parametrize("kind", sorted(WEIGHTS))
@pytest.mark.parametrize("lens,keep,n_sink,n_recent", [
    ([0, 1, 2, 9], 2, 0, 0), ([5, 700, 64], 64, 4, 16), ([257, 1500], 256, 0, 256), ([1030], 1024, 3, 1020), ([3000, 511], 500, 0, 0),
    ([4097, 20], 1, 0, 0), ([130], 129, 1, 1)])
def test_select(kind, lens, keep, n_sink, n_recent):
    kv = KVCache.new_int4(2, 3, 64, max(lens) + 5, len(lens))
    for s, m in enumerate(lens):
        kv.set_seq_len(m, s)
    w = WEIGHTS[kind]((2, len(lens), 3, max(lens) + 5))
    got = kv.select_slots(w.cuda(), keep, n_sink, n_recent)
    assert torch.equal(got.cpu(), chosen(w, lens, keep, n_sink, n_recent))


@pytest.mark.parametrize("n,keep", [(20000, 4096), (33000, 1), (70001, 60000), (16384, 16383), (131072, 8000)])
def test_select_of_long_sequences(n, keep):
    kv = KVCache.new_int4(1, 2, 8, n, 1)
    kv.set_seq_len(n)
    for kind in ("normal", "ties", "zeros"):
        w = WEIGHTS[kind]((1, 1, 2, n))
        want = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
        assert torch.equal(kv.select_slots(w.cuda(), keep).cpu().long(), want), kind


def picked(lens, n_layers, n_kv, keep, seed):
    """Ascending slots, drawn, -1 behind a shorter sequence's last."""
    g = torch.Generator().manual_seed(seed)
    out = torch.full((n_layers, len(lens), n_kv, keep), -1, dtype=torch.int32)
    for s, n in enumerate(lens):
        for i in range(n_layers):
            for h in range(n_kv):
                at = torch.randperm(n, generator=g)[:keep].sort().values
                out[i, s, h, :len(at)] = at.to(torch.int32)
    return out


KEEPS = [([0, 1, 70], 33, 4, 64), ([300, 64, 65], 64, 2, 128), ([200], 31, 3, 256), ([1000, 500], 700, 2, 80), ([129, 128], 128, 2, 40),
         ([95], 94, 1, 8), ([2000], 1999, 2, 96), ([640, 63], 1, 2, 128), ([77, 40], 100, 2, 64), ([1500], 1000, 2, 256)]


def rows_of(kv, lens):
    return [[tuple(x.clone() for x in p) if p else None for p in cached(kv, i, lens)] for i in range(kv.n_layers)]


def check_rows(got, before, slots, lens, keep):
    for i, layer in enumerate(got):
        for s, pair in enumerate(layer):
            n = min(lens[s], keep)
            for h in range(slots.shape[2]):
                at = slots[i, s, h, :n].long()
                for x, y in zip(pair or (), before[i][s] or ()):
                    assert torch.equal(x[:, h], y[at, h]), (i, s, h)


@pytest.mark.parametrize("lens,keep,n_kv,hd", KEEPS)
def test_keep_in_place(lens, keep, n_kv, hd):
    L, cap = 2, max(lens) + 40
    kv = cache(lens, L, n_kv, hd, cap, seed=3)
    before, slots = rows_of(kv, lens), picked(lens, L, n_kv, keep, 5)
    w = rand((L, len(lens), n_kv, cap), 7)
    for s, m in enumerate(lens):
        w[:, s, :, m:] = 0
    dev = w.cuda()
    kv.keep_slots(slots.cuda(), dev)
    kept = [min(m, keep) for m in lens]
    assert kv.seq_lens() == kept and [kv.get_window_base(s) for s in range(len(lens))] == [m - n for m, n in zip(lens, kept)]
    check_rows(rows_of(kv, kept), before, slots, lens, keep)
    for s, n in enumerate(kept):
        for i in range(L):
            for h in range(n_kv):
                want = torch.zeros(cap)
                want[:n] = w[i, s, h, slots[i, s, h, :n].long()]
                assert torch.equal(dev[i, s, h].cpu(), want)
    # the rows append goes on with
    rope = RopeTable.scaled(max(lens) + 1, hd, BASE)
    k = rand((len(lens), 1, n_kv, hd), 8)
    for i in range(L):
        kv.append_quant(i, k.cuda(), k.cuda(), rope)
    check_rows([[tuple(x[:n] for x in p) if n else None for p, n in zip(layer, kept)] for layer in rows_of(kv, [n + 1 for n in kept])],
               before, slots, lens, keep)


@pytest.mark.parametrize("lens,keep,n_kv,hd", KEEPS)
@pytest.mark.parametrize("same", [False, True])
def test_keep_elsewhere(lens, keep, n_kv, hd, same):
    """Sequences 1 .. of a cache into sequences behind them, of another cache or of the same; all others as they were."""
    L, n = 2, len(lens)
    full = [9, *lens] + ([max(lens)] * n + [5] if same else [])
    src = cache(full, L, n_kv, hd, max(lens) + 9, seed=4)
    dst = src if same else cache([17] * (n + 3), L, n_kv, hd, keep + 25, seed=30)
    seq = n + 1 if same else 2
    others = [s for s in range(dst.n_seq) if not seq <= s < seq + n]
    lens_before = dst.seq_lens()
    was, before = rows_of(dst, lens_before), rows_of(src, src.seq_lens())
    slots = picked(lens, L, n_kv, keep, 6)
    sw = rand((L, src.n_seq, n_kv, src.max_seq_len), 9).cuda()
    dw = sw if same else torch.full((L, dst.n_seq, n_kv, dst.max_seq_len), 7.0, device="cuda")
    old = dw.cpu().clone()
    dst.keep_slots(slots.cuda(), dw, src=src, src_weights=sw, seq=seq, src_seq=1, n_seq=n)
    kept = [min(m, keep) for m in lens]
    ends = dst.seq_lens()
    assert ends[seq:seq + n] == kept and [ends[s] for s in others] == [lens_before[s] for s in others]
    assert [dst.get_window_base(seq + s) for s in range(n)] == [m - c for m, c in zip(lens, kept)]
    now = rows_of(dst, ends)
    check_rows([layer[seq:seq + n] for layer in now], [layer[1:1 + n] for layer in before], slots, lens, keep)
    for s in others:
        for i in range(L):
            if was[i][s]:
                assert torch.equal(now[i][s][0], was[i][s][0]) and torch.equal(now[i][s][1], was[i][s][1])
    got = dw.cpu()
    for i in range(L):
        for h in range(n_kv):
            for s in others:
                assert torch.equal(got[i, s, h], old[i, s, h])
            for s, c in enumerate(kept):
                want = torch.zeros(dst.max_seq_len)
                want[:c] = (old if same else sw.cpu())[i, 1 + s, h, slots[i, s, h, :c].long()]
                assert torch.equal(got[i, seq + s, h], want)


@pytest.mark.parametrize("hd", [64, 128, 96])
def test_weigh_evict_and_go_on(hd):
    """A run: chunks and tokens weighed, the cache cut, more tokens; the attention after the cut is that over the kept rows."""
    lens, n_kv, heads, keep, L = [300, 90], 2, 8, 100, 2
    rope = RopeTable.scaled(500, hd, BASE)
    kv = cache(lens, L, n_kv, hd, 400, seed=1, rope=rope)
    w = kv.new_weights()
    q = rand((2, 8, heads, hd), 20, scale=2.0)
    for i in range(L):
        kv.append_quant(i, rand((2, 8, n_kv, hd), 21 + i).cuda(), rand((2, 8, n_kv, hd), 23 + i).cuda(), rope)
        kv.attn_weigh(i, q.cuda(), rope, w[i])
    kv.increment(8)
    ends = [m + 8 for m in lens]
    before = rows_of(kv, ends)
    wc = w.cpu()
    slots = kv.evict(w, keep, n_sink=2, n_recent=10).cpu()
    assert torch.equal(slots, chosen(wc, ends, keep, 2, 10))
    kept = [min(m, keep) for m in ends]
    check_rows(rows_of(kv, kept), before, slots, ends, keep)
    bases = [m - n for m, n in zip(ends, kept)]
    for step in range(3):
        q1 = rand((2, 1, heads, hd), 40 + step, scale=2.0)
        now = [n + step for n in kept]
        for i in range(L):
            old = w[i].cpu()
            k, v = (rand((2, 1, n_kv, hd), 50 + 10 * step + 2 * i + j).cuda() for j in (0, 1))
            out = kv.attn_weigh(i, q1.cuda(), rope, w[i], k=k, v=v)
            want, far, weights = weigh(cached(kv, i, [n + 1 for n in now]), q1, now, bases, hd, hd, BASE)
            assert bool(((out.cpu().double() - want).abs() <= far).all())
            for s, (ws, ws_far) in enumerate(weights):
                n = now[s] + 1
                d = (w[i, s, :, :n].cpu().double() - old[s, :, :n].double() - ws).abs()
                assert bool((d <= ws_far + 2.0 ** -23 * (ws + old[s, :, :n].double())).all())
                assert not bool(w[i, s, :, n:].any())
        kv.increment()
    # the other entry points go on from there too
    alone = kv.attn_decode(0, q1[:, 0].cuda(), rope, out=None)
    assert alone.shape == (2, heads, hd) and bool(torch.isfinite(alone).all())


def test_some_sequences_in_place():
    """Two sequences of four cut, three times over; the others' rows, weights, lengths and bases as they were."""
    lens, L, n_kv, hd, keep, cap = [90, 300, 131, 64], 2, 2, 128, 120, 300
    kv = cache(lens, L, n_kv, hd, cap, seed=31)
    w = rand((L, 4, n_kv, cap), 32).abs()
    for s, m in enumerate(lens):
        w[:, s, :, m:] = 0
    dev = w.cuda()
    for keep in (120, 119, 65):
        before, old, now = rows_of(kv, lens), dev.cpu(), [lens[0], min(lens[1], keep), min(lens[2], keep), lens[3]]
        slots = picked(lens[1:3], L, n_kv, keep, keep)
        kv.keep_slots(slots.cuda(), dev, seq=1, src_seq=1, n_seq=2)
        assert kv.seq_lens() == now and [kv.get_window_base(s) for s in range(4)] == [0, 300 - now[1], 131 - now[2], 0]
        after = rows_of(kv, now)
        for i in range(L):
            for s in (0, 3):
                assert all(torch.equal(x, y) for x, y in zip(after[i][s], before[i][s]))
                assert torch.equal(dev[i, s].cpu(), old[i, s])
            for s in (1, 2):
                for h in range(n_kv):
                    want = torch.zeros(cap)
                    want[:now[s]] = old[i, s, h, slots[i, s - 1, h, :now[s]].long()]
                    assert torch.equal(dev[i, s, h].cpu(), want)
        check_rows([layer[1:3] for layer in after], [layer[1:3] for layer in before], slots, lens[1:3], keep)
        lens = now


def test_more_rows_than_one_launch_takes():
    """12.6 million rows in six slices: 4.8e9 work-items, where a launch takes 2^32, 21 layers of them."""
    n_layers, n_seq, heads, hd = 24, 32768, 16, 8
    rope = RopeTable.scaled(8, hd, 10000.0)
    kv = KVCache.new_int4(n_layers, heads, hd, 3, n_seq)
    w = torch.rand((n_layers, n_seq, heads, 3), device="cuda")
    k = torch.rand((n_seq, 3, heads, hd), device="cuda")
    some = (0, 1, 16, 23)  # layers of either launch
    for i in some:
        kv.append_quant(i, k + i, k - i, rope)
    kv.increment(3)
    off = [3 * s for s in range(n_seq + 1)]
    before = {i: [x.view(n_seq, 3, heads, hd) for x in kv.read_packed(i, off)] for i in some}
    wc = w.clone()
    slots = kv.evict(w, 2)
    # (of equal weights the lowest slots stay: the last of the smallest goes)
    lowest = torch.where(wc == wc.amin(-1, keepdim=True), torch.arange(3, device="cuda"), -1).amax(-1, keepdim=True)
    want = torch.arange(2, device="cuda").expand(slots.shape)
    want = want + (want >= lowest)
    assert torch.equal(slots.long(), want)
    assert torch.equal(w[..., :2], wc.gather(-1, want)) and not bool(w[..., 2].any())
    assert kv.seq_lens() == [2] * n_seq
    off = [2 * s for s in range(n_seq + 1)]
    for i in some:
        at = want[i].transpose(1, 2)[..., None].expand(n_seq, 2, heads, hd)
        for old, new in zip(before[i], kv.read_packed(i, off)):
            assert torch.equal(new.view(n_seq, 2, heads, hd), old.gather(1, at))


def test_weights_of_their_own_in_place():
    """In place with another array for the kept weights: whole rows of it are written."""
    lens, keep = [90, 30], 40
    kv = cache(lens, 2, 2, 64, 120)
    w, to = rand((2, 2, 2, 120), 1).cuda(), torch.full((2, 2, 2, 120), 5.0, device="cuda")
    slots = picked(lens, 2, 2, keep, 2)
    kv.keep_slots(slots.cuda(), to, src_weights=w)
    for i in range(2):
        for s, n in enumerate([40, 30]):
            for h in range(2):
                want = torch.zeros(120)
                want[:n] = w[i, s, h].cpu()[slots[i, s, h, :n].long()]
                assert torch.equal(to[i, s, h].cpu(), want)


def test_captured_choice():
    """select_slots in a graph reads the lengths and weights of its replays."""
    kv = KVCache.new_int4(1, 2, 64, 5000, 2)
    for s, m in enumerate([3000, 50]):
        kv.set_seq_len(m, s)
    w, out = kv.new_weights(), torch.empty((1, 2, 2, 64), dtype=torch.int32, device="cuda")
    kv.select_slots(w, 64, 2, 4, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.select_slots(w, 64, 2, 4, out=out)
    for i, lens in enumerate(([3000, 50], [4900, 700], [64, 4100])):
        for s, m in enumerate(lens):
            kv.set_seq_len(m, s)
        w.copy_(rand(w.shape, 70 + i).cuda())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), chosen(w.cpu(), lens, 64, 2, 4))


def test_another_stream():
    kv = cache([400, 30], 1, 2, 128)
    w, st = rand((1, 2, 2, 400), 1).cuda(), torch.cuda.Stream()
    before = rows_of(kv, [400, 30])
    st.wait_stream(torch.cuda.current_stream())
    wc = w.cpu()
    slots = kv.evict(w, 50, 1, 5, stream=st)
    st.synchronize()
    assert torch.equal(slots.cpu(), chosen(wc, [400, 30], 50, 1, 5))
    check_rows(rows_of(kv, [50, 30]), before, slots.cpu(), [400, 30], 50)


def test_refusals():
    kv, other = cache([50, 20], 2, 2, 64), KVCache.new_int4(2, 2, 64, 16, 2)
    w, ow = kv.new_weights(), other.new_weights()

    def refused(code, call, *a, **k):
        with pytest.raises(TsError) as e:
            call(*a, **k)
        assert e.value.code == code

    for keep, sink, recent in ((0, 0, 0), (-1, 0, 0), (51, 0, 0), (8, 9, 0), (8, 4, 5), (8, -1, 0), (8, 0, -1)):
        refused(-1, kv.select_slots, w, keep, sink, recent)
    with pytest.raises(ValueError):
        kv.select_slots(w[0], 8)
    with pytest.raises(ValueError):
        kv.select_slots(w, 8, out=torch.zeros(2, 2, 2, 9, dtype=torch.int32, device="cuda"))
    slots = kv.select_slots(w, 8)
    with pytest.raises(ValueError):
        kv.keep_slots(slots[:1])
    with pytest.raises(ValueError):
        kv.keep_slots(slots.long())
    with pytest.raises(ValueError):
        other.keep_slots(slots, ow, src=kv)
    refused(-1, kv.keep_slots, slots[:, :1].contiguous(), seq=1, src_seq=2, n_seq=1)
    refused(-1, other.keep_slots, slots, src=kv, seq=1)
    refused(-1, KVCache.new_int4(2, 2, 128, 16, 2).keep_slots, slots, src=kv)
    refused(-1, cache([50, 20, 4], 2, 2, 64).keep_slots, torch.zeros(2, 2, 2, 8, dtype=torch.int32, device="cuda"), seq=1, n_seq=2)  # one of them twice
    many = kv.select_slots(w, 30)
    refused(-2, other.keep_slots, many, src=kv)  # 20 slots into 16
    kv.shift_int4(0, 2, 4)  # a sequence with sinks
    refused(-1, kv.keep_slots, slots)
    kv.reset()
    for s, m in enumerate((50, 20)):
        kv.set_seq_len(m, s)
    kv.keep_slots(slots[:, :0].contiguous(), n_seq=0)  # no sequence: nothing happens
    kv.keep_slots(slots, w)
    assert kv.seq_lens() == [8, 8]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(TsError):
            kv.keep_slots(slots)
        w.zero_()
    assert kv.seq_lens() == [8, 8]
