"""attn_shared against softmax attention in 64 bits over what both caches hold, and against the same
sequences in one unshared cache."""
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import KVCache, RopeTable
from airframe_amd.prompt import attn_prompt, rope_apply
from tests.packed_util import attend, offsets, rand, rope_angles, rotate

pytestmark = pytest.mark.gpu
BASE = 10000.0


class Batch:
    """A prefix of `prefix` positions in sequence prefix_seq of a cache, and a batch behind it."""

    def __init__(self, prefix, own, n_tok, heads, n_kv, hd, prefix_seq=0, norm=False, slack=3, seed=0):
        self.n_seq, self.n_tok, self.heads, self.n_kv, self.hd, self.P = len(own), n_tok, heads, n_kv, hd, prefix
        self.own, self.seq = own, prefix_seq
        self.rope = RopeTable(prefix + max(own) + n_tok + max(slack, 8), hd, BASE)
        self.pre = KVCache.new_int4(2, n_kv, hd, prefix + slack, prefix_seq + 1)
        self.kv = KVCache.new_int4(2, n_kv, hd, max(own) + n_tok + slack, self.n_seq)
        self.qn = self.kn = None
        if norm:
            self.qn, self.kn = (rand((hd,), 70 + i).abs() + 0.5 for i in (0, 1))
            for c in (self.pre, self.kv):
                c.set_qk_norm(1, self.qn.cuda(), self.kn.cuda())
        one = offsets([prefix if s == prefix_seq else 0 for s in range(prefix_seq + 1)])
        self.pk, self.pv = rand((prefix, n_kv, hd), seed + 1), rand((prefix, n_kv, hd), seed + 2)
        self.pre.append_packed(1, self.pk.cuda(), self.pv.cuda(), one, self.rope)
        self.pre.increment_packed(one)
        self.kv.share_prefix(self.pre, prefix_seq)
        off = offsets(own)
        self.k, self.v = rand((off[-1], n_kv, hd), seed + 3), rand((off[-1], n_kv, hd), seed + 4)
        if off[-1]:
            self.kv.append_packed(1, self.k.cuda(), self.v.cuda(), off, self.rope)
            self.kv.increment_packed(off)
        self.nk, self.nv = (rand((self.n_seq, n_tok, n_kv, hd), seed + i) for i in (5, 6))
        self.q = rand((self.n_seq, n_tok, heads, hd), seed + 7)

    def append(self):
        self.kv.append_quant(1, self.nk.cuda(), self.nv.cuda(), self.rope)

    def want(self, softcap=0.0, lens=None):
        """In 64 bits, from the values the caches hold."""
        lens = lens or self.own
        n_pre = self.seq + 1
        pk, pv = (x.cpu() for x in self.pre.read_packed(1, offsets([self.P if s == self.seq else 0 for s in range(n_pre)])))
        angles = rope_angles(self.rope.n_pos, self.hd, BASE)
        out = torch.zeros(self.n_seq, self.n_tok, self.heads, self.hd, dtype=torch.float64)
        g = self.heads // self.n_kv
        for s, m in enumerate(lens):
            n = m + self.n_tok
            k, v = (x.cpu() for x in self.kv.read_packed(1, offsets([n if i == s else 0 for i in range(self.n_seq)])))
            q = self.q[s].double()
            if self.qn is not None:
                q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + 1e-6) * self.qn.double()
            pos = self.P + m + torch.arange(self.n_tok)
            q = rotate(q, angles[pos].cos(), angles[pos].sin(), "interleaved")
            hidden = torch.arange(self.P + n)[None] > pos[:, None]
            for h in range(self.heads):
                out[s, :, h] = attend(q[:, h], torch.cat([pk[:, h // g], k[:, h // g]]), torch.cat([pv[:, h // g], v[:, h // g]]),
                                      hidden, softcap)
        return out


def near(got, want, b):
    """Codes times scales are exact in 64 bits up to the read's one rounding (2^-24).  The operator rounds:
    the f32 table (its angles up to 2^-24 n_pos off) and the rotation, q to 22 bits, f32 dots, scales
    and exp2: scores off by at most D = sqrt(hd) Q K (2^-24 n_pos + 2^-20) (Q, K: norms' bound by the largest
    element; rows of unit variance stay below 5), so the output by V (exp(2 D) - 1) at the very most;
    p v to 22 bits and f32 sums over n keys V (2^-20 + n 2^-24)."""
    big = float(max(b.pv.abs().max(), b.nv.abs().max(), 1.0))
    n = b.P + max(b.own) + b.n_tok
    spread = 5.0 if b.qn is None else 8.0
    d = spread * (2.0 ** -24 * b.rope.n_pos + 2.0 ** -20) * b.hd ** 0.5
    tol = big * ((torch.exp(torch.tensor(2 * d)).item() - 1) + 2.0 ** -20 + n * 2.0 ** -24)
    err = (got.cpu().double() - want).abs().max().item()
    assert err <= tol, (err, tol)


CASES = [(1, [0], 1, 1, 64), (63, [0, 5, 64], 4, 2, 64), (64, [1, 200], 8, 2, 128), (700, [3, 0, 31, 90, 17], 12, 4, 80),
         (333, [64, 2], 5, 1, 256), (1500, [7] * 20, 8, 1, 128), (130, [12, 400], 24, 2, 200), (257, [33] * 3, 16, 1, 64)]


@pytest.mark.parametrize("softcap,norm", [(0.0, False), (5.0, False), (0.0, True)])
@pytest.mark.parametrize("n_tok", [1, 3, 70])
@pytest.mark.parametrize("prefix,own,heads,n_kv,hd", CASES)
def test_shared(gpu, prefix, own, heads, n_kv, hd, n_tok, softcap, norm):
    b = Batch(prefix, own, n_tok, heads, n_kv, hd, norm=norm)
    b.append()
    got = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap)
    near(got, b.want(softcap), b)
    assert torch.equal(got, b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap))


@pytest.mark.parametrize("prefix,own,heads,n_kv,hd", CASES)
def test_shared_appends(gpu, prefix, own, heads, n_kv, hd):
    """The fused append writes what append_quant writes, and the outputs agree."""
    b, c = (Batch(prefix, own, 1, heads, n_kv, hd, prefix_seq=2) for _ in range(2))
    b.append()
    got = c.kv.attn_shared(1, c.q.cuda(), c.rope, c.pre, 2, k=c.nk.cuda(), v=c.nv.cuda())
    for s, m in enumerate(own):
        assert all(torch.equal(x, y) for x, y in zip(b.kv.export(1, s, 0, m + 1), c.kv.export(1, s, 0, m + 1)))
    near(got, b.want(), b)


@pytest.mark.parametrize("heads,n_kv,hd", [(8, 2, 128), (4, 1, 256), (32, 8, 64)])
def test_shared_long_prefix(gpu, heads, n_kv, hd):
    """A prefix in many pieces, few rows."""
    b = Batch(9000, [5, 130], 1, heads, n_kv, hd)
    b.append()
    near(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre), b.want(), b)


@pytest.mark.parametrize("n_tok", [2, 9])
@pytest.mark.parametrize("own", [[900, 3, 0, 517], [1400]])
def test_shared_pieces_of_own_keys(gpu, own, n_tok):
    """A few tokens over long own keys, in pieces that shorter sequences have nothing in."""
    b = Batch(200, own, n_tok, 8, 2, 128)
    b.append()
    near(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre), b.want(), b)


def test_shared_equals_unshared(gpu):
    """A whole run: prompts behind a prefix, a chunk and then tokens, against one cache per sequence that
    holds prefix and all; the packed operators feed both."""
    P, own, heads, n_kv, hd = 150, [20, 7, 33], 8, 2, 64
    rope = RopeTable(400, hd, BASE)
    g = lambda n, h, i: rand((n, h, hd), i).cuda()  # noqa: E731
    pk, pv = g(P, n_kv, 1), g(P, n_kv, 2)
    off = offsets(own)
    k, v = g(off[-1], n_kv, 3), g(off[-1], n_kv, 4)
    pre, kv = KVCache.new_int4(1, n_kv, hd, P), KVCache.new_int4(1, n_kv, hd, 64, 3)
    whole = KVCache.new_int4(1, n_kv, hd, 256, 3)
    pre.append_packed(0, pk, pv, [0, P], rope)
    pre.increment_packed([0, P])
    kv.share_prefix(pre)
    for c, batch in ((kv, [(k, v, off)]), (whole, [(pk.repeat(3, 1, 1), pv.repeat(3, 1, 1), offsets([P] * 3)), (k, v, off)])):
        for bk, bv, o in batch:
            c.append_packed(0, bk, bv, o, rope)
            c.increment_packed(o)
    for step, n_tok in enumerate((5, 1, 1)):
        nk, nv = (rand((3, n_tok, n_kv, hd), 10 * step + i).cuda() for i in (5, 6))
        q = rand((3, n_tok, heads, hd), 10 * step + 7).cuda()
        for c in (kv, whole):
            c.append_quant(0, nk, nv, rope)
        got = kv.attn_shared(0, q, rope, pre)
        want = whole.attn_prefill(0, q, rope) if n_tok > 1 else whole.attn_decode(0, q[:, 0], rope)[:, None]
        # both within near()'s bound of the same 64-bit result: 2^-20 (5 sqrt(64)) 2 4.5 each
        assert (got - want).abs().max() <= 2 * 4.5 * (2 * 40 * (2.0 ** -20) + 2.0 ** -19)
        for c in (kv, whole):
            c.increment(n_tok)
    # the prompts' own attention over what the cache holds, through the packed operators: the last prompt
    # token of each sequence, over the whole cache read back, is its decode
    lens = whole.seq_lens()
    wo = offsets(lens)
    hk, hv = whole.read_packed(0, wo)
    q = rand((wo[-1], heads, hd), 99).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    full = attn_prompt(rope_apply(q, pos, rope), hk, hv, wo)
    last = torch.tensor(wo[1:]).cuda() - 1
    for s in range(3):
        whole.set_seq_len(lens[s] - 1, s)
    dec = whole.attn_decode(0, q[last].contiguous(), rope)
    assert (full[last] - dec).abs().max() <= 2 * 4.5 * (2 * 40 * (2.0 ** -20) + 2.0 ** -19)


def test_shared_no_prefix(gpu):
    """A prefix of no positions is none."""
    b = Batch(4, [5, 0], 1, 4, 2, 64)
    empty = KVCache.new_int4(2, 2, 64, 8)
    b.append()
    b.kv.reset()
    b.kv.append_quant(1, b.nk.cuda(), b.nv.cuda(), b.rope)
    got = b.kv.attn_shared(1, b.q.cuda(), b.rope, empty)
    assert torch.equal(got[:, 0], b.kv.attn_decode(1, b.q[:, 0].contiguous().cuda(), b.rope))


def test_shared_compacted_window(gpu):
    """Own keys compacted behind the prefix (keep_sink 0): the tokens still see the prefix at its place
    and their window at the compacted distance."""
    b = Batch(90, [40, 25], 1, 4, 2, 64)
    b.kv.compact(0, 16, seq=0)
    assert b.kv.seq_lens() == [24, 25] and b.kv.get_window_base(0) == 106
    b.append()
    got = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)
    # sequence 0: its keys moved down, rotated as before; the query sits at 106 + 24 = 90 + 40
    pk, pv = (x.cpu() for x in b.pre.read_packed(1, [0, 90]))
    k, v = (x.cpu() for x in b.kv.read_packed(1, [0, 25, 25]))
    a = rope_angles(b.rope.n_pos, 64, BASE)
    q = rotate(b.q[0].double(), a[130:131].cos(), a[130:131].sin(), "interleaved")
    want = torch.stack([attend(q[:, h], torch.cat([pk[:, h // 2], k[:, h // 2]]), torch.cat([pv[:, h // 2], v[:, h // 2]]),
                               torch.zeros(1, 115, dtype=torch.bool)) for h in range(4)], 1)
    near(got[:1], want[None], b)


@pytest.mark.parametrize("n_tok", [1, 6])
def test_shared_what_lies_behind(gpu, n_tok):
    """Infinities left in slots behind a prefix that was shortened, and (chunks) in a later token of the
    same chunk, reach nobody that does not see them."""
    b = Batch(100, [9, 30], n_tok, 4, 2, 64, slack=40)
    b.append()
    want = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)
    bad = torch.full((20, 2, 64), float("inf"), device="cuda")
    b.pre.append_packed(1, bad, bad, [0, 20], b.rope)
    assert torch.equal(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre), want)
    # and in slots of the batch's own, behind what it holds
    kept = b.kv.seq_lens()
    b.kv.increment(n_tok)
    bad = torch.full((2, 20, 2, 64), float("inf"), device="cuda")
    b.kv.append_quant(1, bad, bad, b.rope)
    for s, m in enumerate(kept):
        b.kv.set_seq_len(m, s)
    assert torch.equal(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre), want)
    if n_tok > 1:
        b.nv[:, 4, :, 3] = float("inf")
        b.append()
        got = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)
        assert torch.equal(got[:, :4], want[:, :4])


@pytest.mark.parametrize("n_tok", [1, 5])
def test_shared_graph(gpu, n_tok):
    """A step captured once: append, attention and lengths, replayed behind each other with eager work
    between, against eager steps."""
    b, c = (Batch(300, [2, 40, 11], n_tok, 8, 2, 128, slack=60) for _ in range(2))
    q, k, v = (torch.zeros_like(x, device="cuda") for x in (b.q, b.nk, b.nv))

    def step(x):
        if n_tok == 1:
            out = x.kv.attn_shared(1, q, x.rope, x.pre, k=k, v=v)
        else:
            x.kv.append_quant(1, k, v, x.rope)
            out = x.kv.attn_shared(1, q, x.rope, x.pre)
        x.kv.increment(n_tok)
        return out

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = step(b)
    for i in range(5):
        for j, x in enumerate((q, k, v)):
            x.copy_(rand(tuple(x.shape), 100 + 10 * i + j).cuda())
        graph.replay()
        c.q, c.nk, c.nv = q.cpu(), k.cpu(), v.cpu()
        got = step(c)
        torch.cuda.synchronize()
        c.own = [m + n_tok * i for m in (2, 40, 11)]
        near(out, c.want(), c)
        assert (out - got).abs().max() <= 2.0 ** -17  # (another split of the same keys)


def test_shared_refusals(gpu):
    b = Batch(20, [3, 4], 1, 4, 2, 64)
    q, k = b.q.cuda(), b.nk.cuda()
    kv, pre, rope = b.kv, b.pre, b.rope
    assert kv.attn_shared(1, q[:, :0].contiguous(), rope, pre).shape == (2, 0, 4, 64)
    for bad in (lambda: kv.attn_shared(1, q[:1], rope, pre), lambda: kv.attn_shared(1, q.half(), rope, pre),
                lambda: kv.attn_shared(1, q, rope, pre, k=k), lambda: kv.attn_shared(1, q, rope, pre, k=k[:1], v=k[:1]),
                lambda: kv.attn_shared(1, q, rope, pre, out=q[:1]), lambda: kv.share_prefix(pre)):
        with pytest.raises(ValueError):
            bad()
    short = torch.zeros(kv.attn_shared_workspace(pre, 4) - 1, dtype=torch.uint8, device="cuda")
    others = [KVCache.new_int4(2, *x) for x in ((1, 64, 8), (2, 128, 8))]
    plain = KVCache.new_int4(2, 2, 64, 8, 2)  # window base 0
    full = KVCache.new_int4(2, 2, 64, 4, 2)
    full.share_prefix(pre)
    full.set_seq_len(4, 1)
    wide = torch.zeros(2, 3, 4, 64, device="cuda")
    for bad, code in ((lambda: kv.attn_shared(2, q, rope, pre), -1), (lambda: kv.attn_shared(1, q, rope, kv), -1),
                      (lambda: kv.attn_shared(1, q, rope, pre, 1), -1), (lambda: kv.attn_shared(1, q, rope, pre, -1), -1),
                      (lambda: kv.attn_shared(1, q[:, :, :3].contiguous(), rope, pre), -1),
                      (lambda: kv.attn_shared(1, q, rope, pre, softcap=-1.0), -1),
                      (lambda: kv.attn_shared(1, q, RopeTable(20, 64, BASE), pre), -1),
                      (lambda: kv.attn_shared(1, q, rope, others[0]), -1), (lambda: kv.attn_shared(1, q, rope, others[1]), -1),
                      (lambda: plain.attn_shared(1, q, rope, pre), -1), (lambda: full.attn_shared(1, q, rope, pre), -2),
                      (lambda: kv.attn_shared(1, wide, rope, pre, k=k, v=k), -1),
                      (lambda: kv.attn_shared(1, q, rope, pre, workspace=short), -6)):
        with pytest.raises(TsError) as e:
            bad()
        assert e.value.code == code


@pytest.mark.parametrize("n_tok", [1, 2, 40])
@pytest.mark.parametrize("heads,n_kv,hd", [(8, 2, 128), (4, 2, 256), (8, 8, 64)])
def test_shared_columns_of_other_scales(gpu, n_tok, heads, n_kv, hd):
    """Sequences whose q is huge, infinite or NaN stand in one matrix product with ordinary ones, which keep
    every bit of their accuracy."""
    b = Batch(300, [40, 3, 0, 11, 25], n_tok, heads, n_kv, hd)
    b.append()
    b.q[0] *= 2.0 ** 30
    b.q[1, :, 0, 5] = float("inf")
    b.q[2] = float("nan")
    got = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)
    assert got[1, :, 0].isnan().all() and got[2].isnan().all() and got[0].isfinite().all()
    near(got[3:], b.want()[3:], b)


def test_shared_compacted_prefix(gpu):
    """A prefix whose own window was compacted ends at its length plus its window base, and the batch goes on
    from there: against one cache that went through the same."""
    rope = RopeTable(400, 64, BASE)
    pk, pv = rand((90, 2, 64), 1).cuda(), rand((90, 2, 64), 2).cuda()
    nk, nv, q = (rand((1, 5, h, 64), i).cuda() for h, i in ((2, 3), (2, 4), (4, 5)))
    pre, kv, whole = KVCache.new_int4(1, 2, 64, 96), KVCache.new_int4(1, 2, 64, 64), KVCache.new_int4(1, 2, 64, 160)
    for c in (pre, whole):
        c.append_packed(0, pk, pv, [0, 90], rope)
        c.increment(90)
        c.compact(4, 20)
    kv.advance_window_base(70)  # (its length alone)
    with pytest.raises(TsError) as e:
        kv.attn_shared(0, q, rope, pre)
    assert e.value.code == -1
    kv.reset()
    kv.share_prefix(pre)
    assert kv.get_window_base() == 90
    for c in (kv, whole):
        c.append_quant(0, nk, nv, rope)
    got, want = kv.attn_shared(0, q, rope, pre), whole.attn_prefill(0, q, rope)
    # both within near()'s bound of the same 64-bit result
    assert (got - want).abs().max() <= 2 * 4.5 * (2 * 40 * (2.0 ** -20) + 2.0 ** -19)
    # own sinks would stand at positions of the prefix
    kv.reset()
    kv.append_quant(0, nk, nv, rope)
    kv.increment(5)
    kv.compact(1, 2)
    kv.advance_window_base(200)
    with pytest.raises(TsError) as e:
        kv.attn_shared(0, q, rope, pre)
    assert e.value.code == -1
