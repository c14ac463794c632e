"""The second status word names the first sequence whose length or pages are out of range, however many there are."""
import pytest
import torch

from cache_helpers import make_cache

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, 64, 16), (torch.float16, 256, 32), (torch.float32, 64, 16), (torch.bfloat16, 33, 7)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,d,page", KINDS)
def test_first_of_many_bad_sequences(dtype, d, page, masked):
    import hbsattn_b200 as hb
    g = torch.Generator().manual_seed(1)
    # more sequences than SMs, so that every CTA walks several of them
    batch, n = 700, 4 * page
    c = make_cache(2, [n] * batch, 2, d, page, dtype, extra_pages=0)
    q = torch.randn(batch, 4, d, generator=g).to(dtype).cuda()
    blocks = -(-n // 16)
    more = dict(block_mask=torch.ones(batch, 2, blocks, dtype=torch.bool, device="cuda"), k_block_size=16) if masked else {}

    def status(lens, table):
        hb.paged_attention(q, c["k"], c["v"], table, lens, **more)
        return hb.last_status()[:2]
    assert status(c["cache_lens"], c["table"]) == [0, 0]
    for first in (0, 1, 2, 3, 350, 699):
        bad = sorted({first, *(torch.randint(first, batch, (40,), generator=g).tolist()), *range(first, min(first + 5, batch))})
        lens = c["cache_lens"].clone()
        lens[bad] = torch.where(torch.rand(len(bad), generator=g) < 0.5, -3, 10 * n).to(torch.int32).cuda()
        assert status(lens, c["table"]) == [3, first]
        table = c["table"].clone()
        table[bad, 1] = -1
        assert status(c["cache_lens"], table) == [3, first]
        if first > 0:                                      # both: a page of a sequence before the lengths
            table = c["table"].clone()
            table[first - 1, 3] = c["k"].shape[0]
            assert status(lens, table) == [3, first - 1]


def test_two_lengths_out_of_range():
    import hbsattn_b200 as hb
    c = make_cache(3, [64] * 4, 2, 64, 16, torch.bfloat16, extra_pages=0)
    q = torch.ones(4, 4, 64, dtype=torch.bfloat16, device="cuda")
    for _ in range(20):
        hb.paged_attention(q, c["k"], c["v"], c["table"], torch.tensor([64, 1000, -3, 64], dtype=torch.int32, device="cuda"))
        assert hb.last_status()[:2] == [3, 1]
