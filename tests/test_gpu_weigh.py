"""attn_weigh against softmax attention in 64 bits over what the cache holds."""
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import KVCache, RopeTable
from tests.evict_util import cached, weigh
from tests.packed_util import offsets, rand

pytestmark = pytest.mark.gpu
BASE = 10000.0


class Batch:
    """A cache whose sequences hold lens[s] slots, and n_tok new tokens of each."""

    def __init__(self, lens, n_tok, heads, n_kv, hd, norm=False, slack=3, seed=0, base=None, rope_dim=None, n_layers=2):
        self.n_seq, self.lens, self.n_tok, self.heads, self.n_kv, self.hd = len(lens), list(lens), n_tok, heads, n_kv, hd
        self.cap = max(lens) + n_tok + slack
        self.base = [base or 0] * self.n_seq
        self.rope_dim = rope_dim or hd
        self.rope = RopeTable.scaled(self.cap + (base or 0), self.rope_dim, BASE)
        self.kv = KVCache.new_int4(n_layers, n_kv, hd, self.cap, self.n_seq)
        self.layer = n_layers - 1
        self.qn = None
        if norm:
            self.qn, kn = (rand((hd,), 70 + i).abs() + 0.5 for i in (0, 1))
            self.kv.set_qk_norm(self.layer, self.qn.cuda(), kn.cuda())
        for s in range(self.n_seq if base else 0):
            self.kv.advance_window_base(base, s)
        off = offsets(lens)
        if off[-1]:
            k, v = rand((off[-1], n_kv, hd), seed + 1), rand((off[-1], n_kv, hd), seed + 2)
            self.kv.append_packed(self.layer, k.cuda(), v.cuda(), off, self.rope)
            self.kv.increment_packed(off)
        self.nk, self.nv = (rand((self.n_seq, n_tok, n_kv, hd), seed + i).cuda() for i in (3, 4))
        self.q = rand((self.n_seq, n_tok, heads, hd), seed + 5, scale=2.0)
        self.w = torch.full((self.n_seq, n_kv, self.cap), float("nan"), device="cuda")

    def append(self):
        self.kv.append_quant(self.layer, self.nk, self.nv, self.rope)

    def check(self, out, w, before=None, softcap=0.0, lens=None):
        lens = lens or self.lens
        ends = [m + self.n_tok for m in lens]
        want, far, weights = weigh(cached(self.kv, self.layer, ends), self.q, lens, self.base, self.hd, self.rope_dim, BASE,
                                   softcap, self.qn)
        off = (out.cpu().double() - want).abs()
        assert bool((off <= far).all()), f"out: {float((off / far).max()):.2f} of the bound"
        w = w.cpu().double()
        for s, (ws, ws_far) in enumerate(weights):
            n = ends[s]
            old = 0.0 if before is None else before[s, :, :n].double()
            d = (w[s, :, :n] - old - ws).abs()
            limit = ws_far + 2.0 ** -23 * (ws + old)
            assert bool((d <= limit).all()), f"weights of {s}: {float((d / limit).max()):.2f} of the bound"
            rest = w[s, :, n:]
            assert torch.equal(rest, torch.zeros_like(rest) if before is None else before[s, :, n:].double())


SHAPES = [
    # lens, n_tok, heads, n_kv, hd
    ([0], 1, 4, 4, 64), ([0, 1, 2], 1, 8, 2, 64), ([63, 64, 65], 1, 32, 8, 64), ([511], 1, 32, 8, 64), ([300, 5], 1, 6, 2, 128),
    ([1500, 0, 77], 1, 32, 8, 128), ([4000], 1, 16, 2, 128), ([129], 1, 9, 1, 64), ([700, 33], 1, 17, 1, 128), ([90, 600], 1, 10, 1, 256),
    ([1300], 1, 16, 8, 256), ([200, 31], 1, 12, 4, 96), ([77], 1, 8, 8, 8), ([250], 1, 4, 2, 40), ([333, 1], 1, 16, 8, 80),
    ([0], 2, 4, 2, 64), ([0], 33, 6, 2, 128), ([5, 64], 3, 32, 8, 128), ([1000, 7, 0], 32, 8, 2, 128), ([63], 130, 4, 1, 64),
    ([400, 100], 65, 3, 3, 256), ([31], 70, 5, 1, 80), ([500], 17, 16, 1, 64), ([2500, 900], 9, 8, 2, 128), ([100], 40, 34, 2, 128),
    ([40, 300, 7, 64], 160, 8, 2, 96), ([0, 130], 257, 4, 1, 128), ([120, 30], 200, 2, 1, 256), ([3000, 2900, 3100, 3050], 330, 16, 8, 64),
]


@pytest.mark.parametrize("lens,n_tok,heads,n_kv,hd", SHAPES)
def test_against_64_bits(lens, n_tok, heads, n_kv, hd):
    b = Batch(lens, n_tok, heads, n_kv, hd, seed=len(SHAPES) + heads)
    b.append()
    out = b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True)
    b.check(out, b.w)
    # added to what is there; slots behind the newest token are left
    before = rand(b.w.shape, 9).abs()
    w = before.cuda()
    again = b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, w)
    b.check(again, w, before)
    assert torch.equal(out, again)
    assert b.kv.seq_lens() == b.lens


@pytest.mark.parametrize("n_tok,heads,n_kv", [(1, 8, 2), (1, 40, 2), (3, 8, 2), (200, 16, 2)])
@pytest.mark.parametrize("m", [5, 63, 333, 1021])
def test_up_to_the_last_slot(m, n_tok, heads, n_kv):
    """The new tokens fill the cache of the longest sequence."""
    b = Batch([m, 1], n_tok, heads, n_kv, 128, slack=0, seed=m)
    b.append()
    b.check(b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True), b.w)


@pytest.mark.parametrize("n_tok", [1, 2])
def test_the_most_query_heads(n_tok):
    """4096 query heads on one kv head; one more head per kv head is refused."""
    b = Batch([70], n_tok, 4096, 1, 16, seed=1)
    b.append()
    b.check(b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True), b.w)
    with pytest.raises(TsError):
        b.kv.attn_weigh_workspace(4097, n_tok)


@pytest.mark.parametrize("n_tok", [1, 5, 140])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_softcap_norm_and_window_base(n_tok, hd):
    for softcap, norm, base, rope_dim in ((20.0, False, None, None), (0.0, True, 37, None), (5.0, True, 1000, 32)):
        b = Batch([150, 70], n_tok, 8, 2, hd, norm=norm, base=base, rope_dim=rope_dim, seed=hd)
        b.append()
        b.check(b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True, softcap=softcap), b.w, softcap=softcap)


@pytest.mark.parametrize("n_tok", [1, 6, 140])
@pytest.mark.parametrize("softcap", [1e-38, 1e-3, 0.7, 1e6, 3e38])
def test_softcaps_large_and_tiny(n_tok, softcap):
    b = Batch([150, 700], n_tok, 8, 2, 128, seed=6)
    b.append()
    b.check(b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True, softcap=softcap), b.w, softcap=softcap)


@pytest.mark.parametrize("lens,heads,n_kv,hd", [([0, 700], 8, 2, 128), ([511], 32, 8, 64), ([64, 3], 20, 2, 64), ([1025], 16, 8, 256),
                                                ([95, 2000], 24, 8, 128), ([128], 12, 4, 96)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_in_the_call(lens, heads, n_kv, hd, norm):
    b = Batch(lens, 1, heads, n_kv, hd, norm=norm, seed=heads)
    out = b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True, k=b.nk, v=b.nv)
    rows = cached(b.kv, b.layer, [m + 1 for m in lens])
    b.append()
    for got, want in zip(rows, cached(b.kv, b.layer, [m + 1 for m in lens])):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    b.check(out, b.w)


@pytest.mark.parametrize("n_tok", [1, 6, 150])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_what_is_not_seen_has_no_part(n_tok, hd):
    """Rows that a shortened sequence left behind, with infinite and NaN scales, change nothing."""
    b = Batch([70, 200], n_tok, 8, 2, hd, slack=80, seed=3)
    ends = [m + n_tok for m in b.lens]
    for s, e in enumerate(ends):
        b.kv.set_seq_len(e, s)
    bad = torch.full((2, 70, 2, hd), float("nan"))
    bad[:, 1::2] = float("inf")
    b.kv.append_quant(b.layer, bad.cuda(), bad.cuda(), b.rope)
    for s, m in enumerate(b.lens):
        b.kv.set_seq_len(m, s)
    b.append()
    out = b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True)
    b.check(out, b.w)


@pytest.mark.parametrize("n_tok", [1, 4, 200])
def test_the_outputs_are_those_of_attention_alone(n_tok):
    b = Batch([900, 130], n_tok, 16, 4, 128, seed=8)
    b.append()
    out = b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True).cpu()
    alone = (b.kv.attn_decode(b.layer, b.q[:, 0].cuda(), b.rope)[:, None] if n_tok == 1
             else b.kv.attn_prefill(b.layer, b.q.cuda(), b.rope)).cpu()
    _, far, _ = weigh(cached(b.kv, b.layer, [m + n_tok for m in b.lens]), b.q, b.lens, b.base, 128, 128, BASE)
    assert bool(((out.double() - alone.double()).abs() <= 2 * far).all())


@pytest.mark.parametrize("n_tok", [1, 7])
def test_another_stream_and_the_workspace_of_the_caller(n_tok):
    b = Batch([600, 64], n_tok, 8, 2, 128, seed=4)
    b.append()
    ws = torch.empty(b.kv.attn_weigh_workspace(8, n_tok), dtype=torch.uint8, device="cuda")
    out, q = torch.empty_like(b.q, device="cuda"), b.q.cuda()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = b.kv.attn_weigh(b.layer, q, b.rope, b.w, fresh=True, out=out, workspace=ws, stream=st)
    st.synchronize()
    assert got.data_ptr() == out.data_ptr()
    b.check(out, b.w)


@pytest.mark.parametrize("n_tok,heads,hd", [(1, 8, 64), (1, 12, 128), (5, 8, 128)])
def test_captured_steps(n_tok, heads, hd):
    """A graph of append, attention and increment, replayed: every replay against the eager call on the cache of its time."""
    lens = [130, 61]
    b = Batch(lens, n_tok, heads, 4, hd, slack=5 * n_tok, seed=5)
    q, w = b.q.cuda(), torch.zeros_like(b.w)
    ws = torch.empty(b.kv.attn_weigh_workspace(heads, n_tok), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)

    def step():
        if n_tok > 1:
            b.append()
        b.kv.attn_weigh(b.layer, q, b.rope, w, k=b.nk if n_tok == 1 else None, v=b.nv if n_tok == 1 else None, out=out, workspace=ws)

    step()
    w.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
        b.kv.increment(n_tok)
    for s, m in enumerate(lens):
        b.kv.set_seq_len(m, s)
    total = torch.zeros_like(w).cpu()
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        now = [m + n_tok * i for m in lens]
        b.check(out, w, total, lens=now)
        total = w.cpu()


@pytest.mark.parametrize("n_tok,heads,n_kv,hd", [(1, 8, 2, 64), (1, 16, 8, 128), (1, 12, 1, 128), (1, 8, 4, 256), (4, 8, 2, 128), (150, 8, 2, 64),
                                                 (40, 32, 8, 256)])
def test_replays_far_past_the_capture(n_tok, heads, n_kv, hd):
    """A graph of attention captured over a few slots and replayed over thousands, and over a few again."""
    lens = [2900, 1700, 40]
    b = Batch(lens, n_tok, heads, n_kv, hd, seed=8)
    b.append()
    q, out = b.q.cuda(), torch.empty_like(b.q, device="cuda")
    ws = torch.empty(b.kv.attn_weigh_workspace(heads, n_tok), dtype=torch.uint8, device="cuda")
    b.kv.attn_weigh(b.layer, q, b.rope, b.w, out=out, workspace=ws)
    for s in range(3):
        b.kv.set_seq_len(20 + s, s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.kv.attn_weigh(b.layer, q, b.rope, b.w, fresh=True, out=out, workspace=ws)
    for now in (lens, [20, 21, 22], lens):
        for s, m in enumerate(now):
            b.kv.set_seq_len(m, s)
        g.replay()
        torch.cuda.synchronize()
        b.check(out, b.w, lens=now)


@pytest.mark.parametrize("n_tok", [1, 7, 140])
def test_a_sequence_with_sinks(n_tok):
    """Sequences that a shift has cut: their keys keep their rotations, the new tokens go on past the window base."""
    b = Batch([300, 90], n_tok, 8, 2, 128, seed=12)
    b.kv.compact(4, 100, 0)
    b.lens[0] -= 100
    b.base[0] += 100
    b.append()
    b.check(b.kv.attn_weigh(b.layer, b.q.cuda(), b.rope, b.w, fresh=True), b.w)


@pytest.mark.parametrize("n_tok", [1, 6])
def test_two_calls_at_once(n_tok):
    """Two caches on two streams, each with a workspace of its own."""
    pair = [Batch([700, 300], n_tok, 8, 2, 128, seed=40 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in pair]
    for b in pair:
        b.append()
    args = [(b.q.cuda(), torch.empty(b.kv.attn_weigh_workspace(8, n_tok), dtype=torch.uint8, device="cuda")) for b in pair]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(5):
        for i, b in enumerate(pair):
            outs[i] = b.kv.attn_weigh(b.layer, args[i][0], b.rope, b.w, fresh=True, workspace=args[i][1], stream=streams[i])
    torch.cuda.synchronize()
    for b, out in zip(pair, outs):
        b.check(out, b.w)


@pytest.mark.parametrize("n_tok", [1, 3])
def test_offsets_past_32_bits(n_tok):
    """The last sequences of a layer of 10 GB."""
    n_seq, cap = 70, 131072
    kv = KVCache.new_int4(1, 8, 128, cap, n_seq)
    rope = RopeTable.scaled(512, 128, BASE)
    lens = [0] * (n_seq - 2) + [77, 300]
    off = offsets(lens)
    kv.append_packed(0, rand((377, 8, 128), 1).cuda(), rand((377, 8, 128), 2).cuda(), off, rope)
    kv.increment_packed(off)
    k, v = (rand((n_seq, n_tok, 8, 128), i).cuda() for i in (3, 4))
    kv.append_quant(0, k, v, rope)
    q, w = rand((n_seq, n_tok, 16, 128), 5, scale=2.0), torch.zeros((n_seq, 8, cap), device="cuda")
    out = kv.attn_weigh(0, q.cuda(), rope, w).cpu()
    ends = [m + n_tok for m in lens]
    want, far, weights = weigh(cached(kv, 0, ends), q, lens, [0] * n_seq, 128, 128, BASE)
    assert bool(((out.double() - want).abs() <= far).all())
    for s in (0, n_seq - 3, n_seq - 2, n_seq - 1):
        ws, ws_far = weights[s]
        got = w[s].cpu().double()
        assert bool(((got[:, :ends[s]] - ws).abs() <= ws_far + 2.0 ** -23 * ws).all()) and not bool(got[:, ends[s]:].any())
    kv.increment(n_tok)
    before, slots = cached(kv, 0, ends), kv.evict(w[None], 40, 1, 2).cpu()
    after = cached(kv, 0, [min(e, 40) for e in ends])
    for s in (n_seq - 2, n_seq - 1):
        for h in range(8):
            at = slots[0, s, h].long()
            assert torch.equal(after[s][0][:, h], before[s][0][at, h]) and torch.equal(after[s][1][:, h], before[s][1][at, h])


def test_refusals():
    b = Batch([20, 8], 1, 8, 2, 64)
    kv, q = b.kv, b.q.cuda()
    b.append()
    ok = dict(fresh=True)
    with pytest.raises(ValueError):
        kv.attn_weigh(1, q[:, 0], b.rope, b.w, **ok)
    with pytest.raises(ValueError):
        kv.attn_weigh(1, q, b.rope, b.w[..., :-1], **ok)
    with pytest.raises(ValueError):
        kv.attn_weigh(1, q, b.rope, b.w.half(), **ok)
    with pytest.raises(ValueError):
        kv.attn_weigh(1, q, b.rope, b.w.cpu(), **ok)
    with pytest.raises(ValueError):
        kv.attn_weigh(1, q, b.rope, b.w, k=b.nk, **ok)
    for bad in (dict(layer=2), dict(layer=-1), dict(softcap=-1.0), dict(softcap=float("inf"))):
        a = dict(layer=1, softcap=0.0)
        a.update(bad)
        with pytest.raises(TsError) as e:
            kv.attn_weigh(a["layer"], q, b.rope, b.w, softcap=a["softcap"], **ok)
        assert e.value.code == -1
    with pytest.raises(TsError) as e:  # heads that are no multiple
        kv.attn_weigh(1, torch.zeros(2, 1, 5, 64, device="cuda"), b.rope, b.w, **ok)
    assert e.value.code == -1
    with pytest.raises(TsError) as e:
        kv.attn_weigh(1, q, b.rope, b.w, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"), **ok)
    assert e.value.code == -6
    with pytest.raises(TsError) as e:  # the output in place of q
        kv.attn_weigh(1, q, b.rope, b.w, out=q, **ok)
    assert e.value.code == -1
    with pytest.raises(TsError) as e:  # a table that ends before the tokens
        kv.attn_weigh(1, q, RopeTable(20, 64, BASE), b.w, **ok)
    assert e.value.code == -1
    kv.set_seq_len(kv.max_seq_len, 0)
    with pytest.raises(TsError) as e:
        kv.attn_weigh(1, q, b.rope, b.w, **ok)
    assert e.value.code == -2
    kv.set_seq_len(20, 0)
    none = kv.attn_weigh(1, torch.zeros(2, 0, 8, 64, device="cuda"), b.rope, b.w, **ok)
    assert none.shape == (2, 0, 8, 64)
    assert bool(torch.isnan(b.w).all())  # nothing was written by any of these
