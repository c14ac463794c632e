"""int64 tables, lengths and positions beyond 32 bits: out of range, as their neighbours within 32 bits are."""
import pytest
import torch

from cache_helpers import make_cache

pytestmark = pytest.mark.gpu

FAR = [2 ** 32, 2 ** 32 + 1, -2 ** 32, torch.iinfo(torch.int64).min]


@pytest.mark.parametrize("far", FAR)
def test_attention_and_append(far):
    import hbsattn_b200 as hb
    c = make_cache(1, [64, 64, 64], 2, 64, 16, torch.bfloat16, extra_pages=0)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    table = c["table"].long()
    table[1, 2] = far
    bad = c["table"].clone()
    bad[1, 2] = -1
    want = hb.paged_attention(q, c["k"], c["v"], bad, c["cache_lens"])
    assert torch.equal(want, hb.paged_attention(q, c["k"], c["v"], table, c["cache_lens"])) and hb.last_status()[:2] == [3, 1]
    lens = torch.tensor([64, 64, far + 5 if far > 0 else far], device="cuda")
    near = torch.tensor([64, 64, 1000 if far > 0 else -1], dtype=torch.int32, device="cuda")
    want = hb.paged_attention(q, c["k"], c["v"], c["table"], near)
    assert torch.equal(want, hb.paged_attention(q, c["k"], c["v"], c["table"], lens)) and hb.last_status()[:2] == [3, 2]
    before = [c["k"].clone(), c["v"].clone()]
    new = torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 1, 2, 3], device="cuda")
    full = torch.tensor([64, 64, 2 ** 32], device="cuda")                    # no room anywhere
    assert hb.append_to_cache(new, new, cu, c["k"], c["v"], c["table"], full).tolist() == [64, 64, 64]
    for t, b in zip((c["k"], c["v"]), before):
        assert torch.equal(t.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("far", FAR)
def test_select_and_compact(far):
    import hbsattn_b200 as hb
    c = make_cache(3, [64, 64], 1, 64, 16, torch.bfloat16, extra_pages=0)
    w = torch.rand(2, 1, 64, generator=torch.Generator().manual_seed(4)).cuda()
    kept, n = hb.select_keys(w, torch.tensor([far, 2 ** 40], device="cuda"), 8)
    assert n.tolist() == [8 if far > 0 else 0, 8]
    kept = torch.tensor([[[1, far + 2, 9]], [[far, 5, 6]]], device="cuda")
    within = torch.tensor([[[1, -1, 9]], [[-1, 5, 6]]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([3, 3], device="cuda")
    k, v = c["k"].clone(), c["v"].clone()
    hb.compact_cache(k, v, c["table"], c["cache_lens"], within, lens)
    hb.compact_cache(c["k"], c["v"], c["table"].long(), c["cache_lens"].long(), kept, lens)
    for t, b in ((c["k"], k), (c["v"], v)):
        assert torch.equal(t.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
