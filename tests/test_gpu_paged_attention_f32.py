"""Attention of one new token over a paged fp32 cache: group sizes, head dimensions and pages around the units of the fp32 kernel, against the
definition in 64 bits, and pages whose size it does not take."""
import pytest
import torch

from cache_helpers import make_cache
from test_gpu_paged_attention import _check, _q, _weights_check

pytestmark = pytest.mark.gpu

LENS = [1, 0, 2, 7, 8, 9, 63, 64, 65, 700, 1029]


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9, 20])
@pytest.mark.parametrize("d", [4, 20, 64, 68, 128, 132, 256])
def test_groups_and_head_dimensions(d, group):
    import hbsattn_b200 as hb
    hk, page = 2, 24
    c = make_cache(11, LENS, hk, d, page, torch.float32, layout="nhd")
    q = _q(12, len(LENS), group * hk, d, torch.float32)
    start = torch.rand(len(LENS), hk, c["table"].shape[1] * page, generator=torch.Generator().manual_seed(13)).cuda()
    w = start.clone()
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w, return_lse=True)
    assert hb.last_status()[0] == 0
    weights, size = _check(q, c, out, lse)
    _weights_check(w, start, weights, d, max(LENS), size)
    assert torch.equal(out, hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"]))


@pytest.mark.parametrize("page", [8, 12, 40, 1, 64])
@pytest.mark.parametrize("k_block", [16, 48, 112])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_and_blocks(d, k_block, page):
    import hbsattn_b200 as hb
    hk, group = 3, 2
    c = make_cache(21, LENS, hk, d, page, torch.float32, layout="hnd")
    q = _q(22, len(LENS), group * hk, d, torch.float32)
    blocks = -(-c["table"].shape[1] * page // k_block)
    mask = (torch.rand(len(LENS), hk, blocks, generator=torch.Generator().manual_seed(23)) < 0.6)
    mask[3] = False
    mask = mask.cuda()
    start = torch.rand(len(LENS), hk, c["table"].shape[1] * page, generator=torch.Generator().manual_seed(24)).cuda()
    w = start.clone()
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], block_mask=mask, k_block_size=k_block, key_weights=w, return_lse=True)
    assert hb.last_status()[0] == 0
    weights, size = _check(q, c, out, lse, mask=mask, k_block=k_block)
    _weights_check(w, start, weights, d, max(LENS), size)
    assert bool((out[3] == 0).all()) and torch.equal(w[3], start[3])
