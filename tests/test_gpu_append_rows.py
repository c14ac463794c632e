"""Appending with cu_seqlens that reach beyond the packed rows: the new lengths count what has been written and nothing else."""
import pytest
import torch

from cache_helpers import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 33)])
@pytest.mark.parametrize("cu,rows,bad", [
    ([0, 5, 30, 32], [(0, 5), (5, 20), (20, 20)], 1),      # the second sequence ends behind the last row
    ([0, 25, 30, 32], [(0, 20), (20, 20), (20, 20)], 0),   # all but the first lie behind it
    ([-4, 3, 9, 20], [(0, 3), (3, 9), (9, 20)], 0),        # the first begins before the first row
    ([0, 3, 9, 20], [(0, 3), (3, 9), (9, 20)], None),
    ([20, 20, 20, 20], [(20, 20)] * 3, None),
])
def test_rows_that_are_not_there_do_not_count(cu, rows, bad, dtype, d):
    import hbsattn_b200 as hb
    total = 20
    c = make_cache(1, [10, 0, 33], 2, d, 16, dtype, room=40)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(total, 2, d, generator=g).to(dtype).cuda() for _ in "kv")
    want = [c["k"].clone(), c["v"].clone()]
    for b, (lo, hi) in enumerate(rows):
        pos = c["lens"][b] + torch.arange(hi - lo, device="cuda")
        for t, new in zip(want, (k, v)):
            t[c["table"][b].long()[pos // 16], pos % 16] = new[lo:hi]
    lens = hb.append_to_cache(k, v, torch.tensor(cu, dtype=torch.int32).cuda(), c["k"], c["v"], c["table"], c["cache_lens"])
    assert lens.tolist() == [n + hi - lo for n, (lo, hi) in zip(c["lens"], rows)]
    assert hb.last_status()[:2] == ([0, 0] if bad is None else [3, bad])
    for got, t in zip((c["k"], c["v"]), want):
        assert torch.equal(got.contiguous().view(torch.uint8), t.contiguous().view(torch.uint8))


def test_lists_that_do_not_ascend_are_reported():
    import hbsattn_b200 as hb
    c = make_cache(3, [5, 9, 0], 2, 64, 16, torch.bfloat16, fill=0.0, room=30)
    k = torch.ones(20, 2, 64, dtype=torch.bfloat16, device="cuda")
    for cu, first in (([0, 12, 4, 20], 1), ([20, 10, 5, 0], 0), ([0, 1, 30, 2], 1)):
        hb.append_to_cache(k, k, torch.tensor(cu, dtype=torch.int32).cuda(), c["k"], c["v"], c["table"], c["cache_lens"])
        assert hb.last_status()[:2] == [3, first]
