"""Key weights are the same bits every time: items go to CTAs in any order, and what a group of warps is doing in one item says nothing about the
next, but neither may show."""
import pytest
import torch

from helpers import make_problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,hq,hk,d,qbs,kbs,causal,dtype", [
    (([400], [150]), 12, 2, 128, 64, 256, False, torch.float16),              # items of one tile to a few, fewer than CTAs
    (([203, 150, 77], [203, 150, 77]), 8, 2, 64, 80, 48, False, torch.float16),
    (([500, 70, 900], [500, 70, 900]), 6, 3, 256, 48, 80, True, torch.bfloat16),
    (([3000, 100, 17, 2000], [3000, 100, 17, 2000]), 16, 4, 64, 16, 16, True, torch.bfloat16),
    (([2000, 2100], [2000, 2100]), 8, 8, 128, 128, 128, True, torch.bfloat16),
])
def test_same_bits_every_time(lens, hq, hk, d, qbs, kbs, causal, dtype):
    import hbsattn_b200 as hb
    pr = make_problem(91, *lens, hq, hk, d, qbs, kbs, causal, dtype, 0.5, None)
    q = 2 * pr["q"]
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], qbs, kbs, causal)
    _, lse = hb.HBSAttention_with_lse(q, pr["k"], pr["v"], *rest)
    want = hb.attention_key_weights(q, pr["k"], lse, *rest)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        differ += (hb.attention_key_weights(q, pr["k"], lse, *rest) != want).sum()
    assert int(differ) == 0
