"""Compaction of few and of many sequences, short and long: the kernel's slices and block sizes, with the weights moved alike."""
import pytest
import torch

from cache_helpers import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,hk,d,budget", [(1, 1, 128, 5000), (2, 8, 64, 1500), (3, 6, 128, 2000), (12, 8, 128, 1100), (5, 2, 40, 1025), (2, 1, 8, 4096), (9, 8, 256, 300)])
def test_sizes(batch, hk, d, budget, dtype):
    import hbsattn_b200 as hb
    page = 32
    lens = [int(x) for x in torch.randint(budget // 2, 3 * budget, (batch,), generator=torch.Generator().manual_seed(31))]
    c = make_cache(32, lens, hk, d, page, dtype, layout="nhd")
    capacity = c["table"].shape[1] * page
    w = torch.rand(batch, hk, capacity, generator=torch.Generator().manual_seed(33)).cuda()
    kept, kept_lens = hb.select_keys(w, c["cache_lens"], budget, 1, 7)
    before = [c["k"].clone(), c["v"].clone()]
    old_w = w.clone()
    hb.compact_cache(c["k"], c["v"], c["table"], c["cache_lens"], kept, kept_lens, key_weights=w)
    table, i = c["table"].long(), torch.arange(capacity, device="cuda")
    for b, n in enumerate(lens):
        m = min(n, budget)
        for h in range(hk):
            src = kept[b, h, :m].long()
            for new, old in zip((c["k"], c["v"]), before):
                got, want = new[table[b][i[:n] // page], i[:n] % page, h], old[table[b][i[:n] // page], i[:n] % page, h]
                assert torch.equal(got[:m], want[src]) and torch.equal(got[m:], want[m:])
            assert torch.equal(w[b, h, :m], old_w[b, h, src]) and not w[b, h, m:n].any() and torch.equal(w[b, h, n:], old_w[b, h, n:])
