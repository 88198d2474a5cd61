"""attn_shared where a chunk fills the chip (a job walks the prefix and then a sequence's own keys and writes
its output, without partials), and every form of it as closely as its roundings allow."""
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import RopeTable
from tests.packed_util import attend_bound, norms, offsets, rand, rope_angles, rotate
from tests.test_gpu_shared import BASE, Batch

pytestmark = pytest.mark.gpu


class Exact(Batch):
    """A Batch whose table has 64-bit angles, its entries rounded once."""

    def __init__(self, prefix, own, n_tok, *a, slack=3, **kw):
        super().__init__(prefix, own, n_tok, *a, slack=slack, **kw)
        self.rope = RopeTable.scaled(self.rope.n_pos, self.hd, BASE)

    def refill(self):
        """(the caches once more, with keys rotated by that table)"""
        one = offsets([self.P if s == self.seq else 0 for s in range(self.seq + 1)])
        self.pre.reset()
        self.kv.reset()
        self.pre.append_packed(1, self.pk.cuda(), self.pv.cuda(), one, self.rope)
        self.pre.increment_packed(one)
        self.kv.share_prefix(self.pre, self.seq)
        off = offsets(self.own)
        if off[-1]:
            self.kv.append_packed(1, self.k.cuda(), self.v.cuda(), off, self.rope)
            self.kv.increment_packed(off)
        return self

    def is_chain(self):
        """Chunks that need no partials need no workspace."""
        return self.kv.attn_shared_workspace(self.pre, self.heads, self.n_tok) == 0


def close(got, b, softcap=0.0, seqs=None, rows=slice(None)):
    """Within eight standard deviations of the operator's roundings, element by element.

    Keys and values are what the caches hold (codes times scales, read back with one rounding of 2^-24).  q is rotated
    in f32 (2^-24 of it, three times), and held to 2^-21 of its largest element (an f16 and two 6-bit terms, uniform:
    0.6 of that), so that a score is off by 2^-21 0.6 Q k, with Q the largest element of q's rows and k the keys' root
    mean square; sums in f32 by 4 2^-24 q k (16 steps of partial sums below sqrt(hd) q k); its scale, softcap's
    tanh and exp2 by 2^-21 of the largest score.  p v is held to 22 bits, sums of n keys and the join of parts in
    f32: 2^-20 of the largest value."""
    got, g = got.cpu().double(), b.heads // b.n_kv
    pk, pv = (x.cpu() for x in b.pre.read_packed(1, offsets([b.P if s == b.seq else 0 for s in range(b.seq + 1)])))
    angles = rope_angles(b.rope.n_pos, b.hd, BASE)
    for s in range(b.n_seq) if seqs is None else seqs:
        m = b.own[s]
        n = m + b.n_tok
        k, v = (x.cpu() for x in b.kv.read_packed(1, offsets([n if i == s else 0 for i in range(b.n_seq)])))
        q = b.q[s].double()
        if b.qn is not None:
            q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + 1e-6) * b.qn.double()
        pos = b.P + m + torch.arange(b.n_tok)
        q = rotate(q, angles[pos].cos(), angles[pos].sin(), "interleaved")[rows]
        keys, values = torch.cat([pk, k]), torch.cat([pv, v])
        hidden = (torch.arange(b.P + n)[None] > pos[:, None])[rows]
        (qm, qr), (km, kr) = norms(q), norms(keys[keys.isfinite().all(-1).all(-1)])
        x = 6 * qr * kr
        d = 2.0 ** -21 * 0.6 * qm * kr + 7 * 2.0 ** -24 * qr * kr + 2.0 ** -21 * (min(x, softcap) if softcap else x)
        for h in range(b.heads):
            want, by_score, _ = attend_bound(q[:, h], keys[:, h // g], values[:, h // g], hidden, softcap)
            tol = 8 * d * by_score + 2.0 ** -20 * float(values.abs().max())
            err = (got[s, rows, h] - want).abs()
            assert (err <= tol).all(), (s, h, float((err / tol).max()), float(err.max()))


# (sequences' own keys, new tokens, heads, kv heads, head dim, prefix) that fill a chip of 256 CUs and more
CHAINS = [([0, 5, 64, 90, 17, 1, 33, 63], 75, 32, 8, 128, 257), ([3] * 6, 97, 32, 8, 64, 130), ([7, 0, 41], 130, 64, 8, 80, 63),
          ([20, 6, 0, 1], 130, 32, 8, 256, 64), ([11] * 33, 31, 32, 8, 200, 1)]


@pytest.mark.parametrize("softcap,norm", [(0.0, False), (5.0, False), (0.0, True)])
@pytest.mark.parametrize("own,n_tok,heads,n_kv,hd,prefix", CHAINS)
def test_chain(gpu, own, n_tok, heads, n_kv, hd, prefix, softcap, norm):
    b = Exact(prefix, own, n_tok, heads, n_kv, hd, norm=norm).refill()
    assert b.is_chain()
    b.append()
    got = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap)
    close(got, b, softcap, seqs=range(0, len(own), 3))
    assert torch.equal(got, b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap))
    # into rows of the caller's, with those around them left as they are
    wide = torch.full((len(own) + 2, n_tok, heads, hd), 7.0, device="cuda")
    b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap, out=wide[1:-1])
    assert torch.equal(wide[1:-1], got) and (wide[0] == 7).all() and (wide[-1] == 7).all()


@pytest.mark.parametrize("own,n_tok,heads,n_kv,hd,prefix", CHAINS)
def test_chain_what_lies_behind(gpu, own, n_tok, heads, n_kv, hd, prefix):
    """Infinities behind a shortened prefix, behind the sequences' keys and in a later token of the chunk reach nobody
    that does not see them; a NaN or infinite q stays in its own row."""
    b = Exact(prefix, own, n_tok, heads, n_kv, hd, slack=40).refill()
    assert b.is_chain()
    b.append()
    want = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)
    bad = torch.full((20, n_kv, hd), float("inf"), device="cuda")
    b.pre.append_packed(1, bad, bad, [0, 20], b.rope)
    b.kv.increment(n_tok)
    bad = torch.full((len(own), 30, n_kv, hd), float("inf"), device="cuda")
    b.kv.append_quant(1, bad, bad, b.rope)
    for s, m in enumerate(own):
        b.kv.set_seq_len(m, s)
    assert torch.equal(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre), want)
    b.nv[:, 20, :, 3] = float("inf")
    b.nk[:, 21, :, 1] = float("nan")
    b.append()
    assert torch.equal(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)[:, :20], want[:, :20])
    q = b.q.cuda()
    q[0, 2], q[1, 0, 1, 3], q[-1, 5] = float("nan"), float("inf"), q[-1, 5] * 2.0 ** 30
    got = b.kv.attn_shared(1, q, b.rope, b.pre)[:, :20]
    touched = torch.zeros(got.shape[:3], dtype=torch.bool, device="cuda")
    touched[0, 2], touched[1, 0, 1], touched[-1, 5] = True, True, True
    assert torch.equal(got[~touched], want[:, :20][~touched])
    assert got[0, 2].isnan().all() and got[1, 0, 1].isnan().all() and got[-1, 5].isfinite().all()


def test_chain_graph(gpu):
    """A chunk captured once (append, attention, lengths), replayed with eager work between."""
    own, n_tok = [0, 5, 64, 90], 66
    b, c = (Exact(200, own, n_tok, 64, 8, 64, slack=4 * 66).refill() for _ in range(2))
    assert b.is_chain()
    q, k, v = (torch.zeros_like(x, device="cuda") for x in (b.q, b.nk, b.nv))

    def step(x):
        x.kv.append_quant(1, k, v, x.rope)
        out = x.kv.attn_shared(1, q, x.rope, x.pre)
        x.kv.increment(n_tok)
        return out

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = step(b)
    for i in range(4):
        for j, x in enumerate((q, k, v)):
            x.copy_(rand(tuple(x.shape), 100 + 10 * i + j).cuda())
        graph.replay()
        got = step(c)
        torch.cuda.synchronize()
        assert torch.equal(out, got)
    c.q, c.own = q.cpu(), [m + 3 * n_tok for m in own]
    close(got, c, seqs=[0, 3])


CASES = [(1, [0], 1, 1, 64), (700, [3, 0, 31, 90, 17], 12, 4, 80), (333, [64, 2], 5, 1, 256), (1500, [7] * 20, 8, 1, 128),
         (130, [12, 400], 24, 2, 200), (9000, [5, 130], 8, 2, 128)]


@pytest.mark.parametrize("softcap,norm", [(0.0, False), (5.0, False), (50.0, True)])
@pytest.mark.parametrize("n_tok", [1, 3, 40])
@pytest.mark.parametrize("prefix,own,heads,n_kv,hd", CASES)
def test_shared_accuracy(gpu, prefix, own, heads, n_kv, hd, n_tok, softcap, norm):
    b = Exact(prefix, own, n_tok, heads, n_kv, hd, norm=norm).refill()
    b.append()
    close(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap), b, softcap, seqs=range(min(5, len(own))))
    if n_tok == 1:
        b.refill()
        got = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap, k=b.nk.cuda(), v=b.nv.cuda())
        close(got, b, softcap, seqs=range(min(5, len(own))))


@pytest.mark.parametrize("n_tok", [1, 2, 40])
@pytest.mark.parametrize("heads,n_kv,hd", [(8, 2, 128), (4, 2, 256), (8, 8, 64)])
def test_shared_accuracy_beside_others(gpu, n_tok, heads, n_kv, hd):
    """Ordinary sequences beside ones whose q is huge, infinite or NaN keep the bits that they have alone."""
    b = Exact(300, [40, 3, 0, 11, 25], n_tok, heads, n_kv, hd).refill()
    b.append()
    b.q[0] *= 2.0 ** 30
    b.q[1, :, 0, 5] = float("inf")
    b.q[2] = float("nan")
    close(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre), b, seqs=[3, 4])


@pytest.mark.parametrize("n_tok,own", [(1, [5, 0, 70]), (3, [5, 0, 70]), (75, [3] * 8)])
def test_shared_output_in_place(gpu, n_tok, own):
    """The output may be q; another overlap of the two, or of the workspace with any of them, is refused."""
    b = Exact(100, own, n_tok, 32, 8, 64).refill()
    b.append()
    assert b.is_chain() == (n_tok == 75)
    want = b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre)
    n = want.numel()
    space = torch.zeros(n + 1024 + b.kv.attn_shared_workspace(b.pre, 32, n_tok) // 4, device="cuda")
    q = space[:n].view(want.shape)
    q.copy_(b.q)
    assert torch.equal(b.kv.attn_shared(1, q, b.rope, b.pre, out=q), want)
    other = torch.zeros_like(want)
    calls = [lambda: b.kv.attn_shared(1, q, b.rope, b.pre, out=space[64:n + 64].view(want.shape)),
             lambda: b.kv.attn_shared(1, space[64:n + 64].view(want.shape), b.rope, b.pre, out=q)]
    if not b.is_chain():
        ws = space[n - 64:].view(torch.uint8)
        calls += [lambda: b.kv.attn_shared(1, q, b.rope, b.pre, out=other, workspace=ws),
                  lambda: b.kv.attn_shared(1, other, b.rope, b.pre, out=q, workspace=ws)]
    for bad in calls:
        with pytest.raises(TsError) as e:
            bad()
        assert e.value.code == -1


@pytest.mark.parametrize("softcap", [1e-39, 1e4, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("n_tok", [1, 3, 75])
def test_shared_softcap_range(gpu, n_tok, softcap):
    b = Exact(200, [40, 0, 3, 11, 64, 1, 2, 9], n_tok, 32, 8, 128).refill()
    b.append()
    close(b.kv.attn_shared(1, b.q.cuda(), b.rope, b.pre, softcap=softcap), b, softcap, seqs=[0, 4])


def test_shared_workspace_not_needed(gpu):
    """Where no workspace is needed, what is passed for one is not looked at."""
    b = Exact(100, [3] * 8, 75, 32, 8, 64).refill()
    b.append()
    assert b.is_chain()
    q = b.q.cuda()
    want = b.kv.attn_shared(1, q, b.rope, b.pre)
    assert torch.equal(b.kv.attn_shared(1, q, b.rope, b.pre, workspace=q.view(-1)[1024:].view(torch.uint8)), want)
