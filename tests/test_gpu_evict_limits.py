"""The limits of keep_slots, as the header states them."""
import pytest
import torch

from airframe_amd import TsError
from airframe_amd.kv_cache import KVCache, RopeTable
from tests.evict_util import cached
from tests.packed_util import rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("elsewhere", [False, True])
def test_more_slots_named_than_fit(elsewhere):
    """Rows of 240000 named slots (4.9e8 in all) of which a cache holds 64: work goes by what there is to move."""
    n_seq, heads, hd, keep = 2, 1024, 8, 240000
    kv = KVCache.new_int4(1, heads, hd, 64, n_seq)
    x = rand((n_seq, 5, heads, hd), 1).cuda()
    kv.append_quant(0, x, x + 1, RopeTable.scaled(64, hd, 10000.0))
    kv.increment(5)
    before = cached(kv, 0, [5, 5])
    slots = torch.full((1, n_seq, heads, keep), -1, dtype=torch.int32, device="cuda")
    slots[..., :5] = torch.arange(5, dtype=torch.int32, device="cuda")
    to = KVCache.new_int4(1, heads, hd, 64, n_seq) if elsewhere else kv
    to.keep_slots(slots, src=kv)
    assert to.seq_lens() == [5, 5]
    for got, want in zip(cached(to, 0, [5, 5]), before):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("elsewhere", [False, True])
def test_the_most_rows(elsewhere):
    """7456540 rows are taken, one more is refused."""
    for n_seq, fits in ((7456540 // 20, True), (7456540 // 20 + 1, False)):
        kv = KVCache.new_int4(1, 20, 8, 1, n_seq)
        slots = torch.zeros((1, n_seq, 20, 1), dtype=torch.int32, device="cuda")
        to = KVCache.new_int4(1, 20, 8, 1, n_seq) if elsewhere else kv
        if fits:
            to.keep_slots(slots, src=kv)
            assert to.get_seq_len(n_seq - 1) == 0
        else:
            with pytest.raises(TsError) as e:
                to.keep_slots(slots, src=kv)
            assert e.value.code == -1
        del kv, to
