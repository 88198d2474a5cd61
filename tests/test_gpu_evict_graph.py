"""Captured steps that go on after a cut: the window bases of a cache that was cut between replays."""
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import KVCache, RopeTable
from tests.evict_util import cached, weigh
from tests.packed_util import offsets, rand

pytestmark = pytest.mark.gpu
BASE = 10000.0
LENS, KEEP, HEADS, N_KV = [130, 61], 40, 8, 2


class Steps:
    """A cache and one kind of step on it, appending n_tok tokens a sequence and attending to all."""

    def __init__(self, kind, hd, n_tok):
        self.kind, self.hd, self.n_tok = kind, hd, n_tok
        self.rope = RopeTable.scaled(400, hd, BASE)
        self.kv = KVCache.new_int4(1, N_KV, hd, 300, 2)
        off = offsets(LENS)
        k, v = (rand((off[-1], N_KV, hd), i).cuda() for i in (1, 2))
        self.kv.append_packed(0, k, v, off, self.rope)
        self.kv.increment_packed(off)
        self.k, self.v = (torch.empty((2, n_tok, N_KV, hd), device="cuda") for _ in range(2))
        self.q, self.out = (torch.empty((2, n_tok, HEADS, hd), device="cuda") for _ in range(2))
        self.w = self.kv.new_weights()
        need = max(self.kv.attn_weigh_workspace(HEADS, n_tok), self.kv.workspace(HEADS).numel() if n_tok == 1 else 0)
        self.x, self.wq, self.wk, self.wv = torch.empty((2, n_tok, 256), device="cuda"), *(
            rand((h * hd, 256), 60 + h, torch.float16, 1 / 16).cuda() for h in (HEADS, N_KV, N_KV + 1))
        self.wv = self.wv[:N_KV * hd].contiguous()
        self.ws = torch.empty(max(need, 1 << 20), dtype=torch.uint8, device="cuda")

    def inputs(self, i):
        for j, t in enumerate((self.k, self.v, self.q, self.x)):
            t.copy_(rand(t.shape, 100 + 10 * i + j).cuda())

    def run(self):
        """One step; the lengths grow."""
        kv, k, v, q, ws = self.kv, self.k, self.v, self.q, self.ws
        flat = lambda t: t.view(-1, *t.shape[2:])  # noqa: E731
        off = [0, self.n_tok, 2 * self.n_tok]
        if self.kind == "weigh":
            kv.attn_weigh(0, q, self.rope, self.w, k=k, v=v, out=self.out, workspace=ws)
        elif self.kind == "weigh_chunk":
            kv.append_quant(0, k, v, self.rope)
            kv.attn_weigh(0, q, self.rope, self.w, out=self.out, workspace=ws)
        elif self.kind in ("decode", "advance"):
            kv.attn_decode_append(0, k, v, q[:, 0], self.rope, out=self.out[:, 0], workspace=ws, advance=self.kind == "advance")
        elif self.kind == "prefill":
            kv.append_quant(0, k, v, self.rope)
            kv.attn_prefill(0, q, self.rope, out=self.out)
        elif self.kind == "packed":
            kv.append_packed(0, flat(k), flat(v), off, self.rope)
            kv.attn_prefill(0, q, self.rope, out=self.out)
        else:
            kv.qkv_append(0, self.x, self.wq, self.wk, self.wv, self.rope, q_out=self.q, workspace=ws)
            kv.attn_prefill(0, q, self.rope, out=self.out)
        if self.kind == "packed":
            kv.increment_packed(off)
        elif self.kind != "advance":
            kv.increment(self.n_tok)


KINDS = [("weigh", 1), ("weigh_chunk", 3), ("weigh_chunk", 40), ("decode", 1), ("advance", 1), ("prefill", 5), ("packed", 3), ("qkv", 1),
         ("qkv", 9)]


@pytest.mark.parametrize("cut", ["evict", "compact"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind,n_tok", KINDS)
def test_replays_after_a_cut(kind, n_tok, hd, cut):
    """A step captured on a cache that was never cut, replayed before and after a cut: new tokens go on at the positions they
    would have had, as those of eager steps do."""
    a, b = Steps(kind, hd, n_tok), Steps(kind, hd, n_tok)
    a.inputs(0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.run()
    lens, bases = list(LENS), [0, 0]
    for s, m in enumerate(lens):  # (capturing counts as a step on the host)
        a.kv.set_seq_len(m, s)
    for i in range(4):
        if i == 2:
            for s, m in enumerate(lens):
                a.kv.set_seq_len(m, s)
            if cut == "evict":
                slots = a.kv.evict(a.w, KEEP, 2, 10)
                b.kv.keep_slots(slots, b.w)
                now = [min(m, KEEP) for m in lens]
            else:
                for x in (a, b):
                    for s in range(2):
                        x.kv.compact(4, 20, s)
                now = [m - 20 for m in lens]
            bases = [m - n for m, n in zip(lens, now)]
            lens = now
            assert a.kv.seq_lens() == b.kv.seq_lens() == lens
        for x in (a, b):
            x.inputs(i)
        g.replay()
        b.run()
        torch.cuda.synchronize()
        ends = [m + n_tok for m in lens]
        rows, want_rows = cached(a.kv, 0, ends), cached(b.kv, 0, ends)
        for got, want in zip(rows, want_rows):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        want, far, _ = weigh(rows, a.q.cpu(), lens, bases, hd, hd, BASE)
        off = (a.out.cpu().double() - want).abs()
        # (the attention calls' common bound; a position wrong by 20 is off by a hundred times that)
        assert bool((off <= 2e-3 + 1e-3 * want.abs()).all()), (i, float(off.max()))
        lens = ends


@pytest.mark.parametrize("kind,n_tok", KINDS)
def test_replays_past_the_table(kind, n_tok):
    """Replays whose positions pass the last row of the call's table take that row."""
    st = Steps(kind, 128, n_tok)
    st.rope = RopeTable.scaled(LENS[0] + n_tok, 128, BASE)
    st.inputs(0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st.run()
    for s in range(2):
        st.kv.set_seq_len(LENS[0] + 30, s)
    for i in range(2):
        st.inputs(i)
        g.replay()
        torch.cuda.synchronize()
        rows = cached(st.kv, 0, [LENS[0] + 30 + (i + 1) * n_tok] * 2)
        assert all(bool(torch.isfinite(x).all()) for r in rows for x in r)
        assert bool(torch.isfinite(st.out).all())


@pytest.mark.parametrize("elsewhere", [False, True])
def test_a_cut_behind_replays_alone(elsewhere):
    """Replays move the lengths past those that the host knows; a cut without set_seq_len takes the device's, for its bases and
    for the host, twice over."""
    st = Steps("weigh", 128, 1)
    st.inputs(0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st.run()
    for s, m in enumerate(LENS):
        st.kv.set_seq_len(m, s)
    lens, bases, small = list(LENS), [0, 0], KVCache.new_int4(1, N_KV, 128, 70, 2)
    for round_ in range(2):
        for i in range(3):
            st.inputs(10 * round_ + i)
            g.replay()
        lens = [m + 3 for m in lens]
        if elsewhere:
            with pytest.raises(TsError) as e:  # (as many slots as the device has, not as the host knows)
                KVCache.new_int4(1, N_KV, 128, lens[1] - 1, 2).keep_slots(st.kv.select_slots(st.w, 100), src=st.kv)
            assert e.value.code == -2
        before = cached(st.kv, 0, lens)
        slots = st.kv.select_slots(st.w, KEEP, 2, 10)
        to = small if elsewhere else st.kv
        to.keep_slots(slots, src=st.kv) if elsewhere else to.keep_slots(slots, st.w)
        now = [min(m, KEEP) for m in lens]
        cut_bases = [b + m - n for b, m, n in zip(bases, lens, now)]
        assert to.seq_lens() == now and [to.get_window_base(s) for s in range(2)] == cut_bases
        after, at = cached(to, 0, now), slots.cpu().long()
        for s in range(2):
            for h in range(N_KV):
                for x, y in zip(after[s], before[s]):
                    assert torch.equal(x[:, h], y[at[0, s, h, :now[s]], h])
        # an eager token on it
        k, v, q = (rand((2, 1, n, 128), 200 + j, scale=2.0) for j, n in enumerate((N_KV, N_KV, HEADS)))
        w = to.new_weights()
        out = to.attn_weigh(0, q.cuda(), st.rope, w[0], k=k.cuda(), v=v.cuda())
        want, far, _ = weigh(cached(to, 0, [n + 1 for n in now]), q, now, cut_bases, 128, 128, BASE)
        assert bool(((out.cpu().double() - want).abs() <= far).all())
        if not elsewhere:
            lens, bases = now, cut_bases
