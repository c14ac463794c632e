"""Decoding over long rows, which several CTAs share: against the definition in 64 bits within bounds that notice a lost tile
(test_paged_bounds_host.py), and on values that say exactly which keys a result has seen, and how often."""
import math

import pytest
import torch

from cache_helpers import make_cache, rows_of
from paged_bounds import chain, lse_bound, out_bound

pytestmark = pytest.mark.gpu

KINDS = [
    # dtype, nhead_q, nhead_k, d, page
    (torch.bfloat16, 8, 1, 64, 64),
    (torch.float16, 8, 1, 64, 16),
    (torch.bfloat16, 8, 1, 128, 64),
    (torch.float16, 16, 2, 128, 48),
    (torch.bfloat16, 20, 1, 128, 16),                # two times 16 heads
    (torch.bfloat16, 4, 1, 256, 64),                 # halves of the columns
    (torch.float16, 36, 1, 256, 32),                 # and chunks
    (torch.float32, 8, 1, 64, 16),
    (torch.float32, 4, 2, 128, 64),
    (torch.float32, 8, 1, 256, 8),
    (torch.bfloat16, 6, 2, 96, 64),
    (torch.bfloat16, 8, 1, 64, 20),                  # the kernel for odd pages
    (torch.float32, 3, 1, 33, 16),
]
IDS = [f"{str(k[0])[6:]}_{k[1]}x{k[2]}_d{k[3]}_p{k[4]}" for k in KINDS]
LENS = [[20000], [20011, 9000, 1, 0, 12345, 64]]


@pytest.mark.parametrize("lens", LENS, ids=["one", "several"])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_long_rows_within_tight_bounds(kind, lens):
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page = kind
    c = make_cache(1, lens, hk, d, page, dtype, fill=0.0)
    q = (2 * torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(2))).to(dtype).cuda()
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], return_lse=True)
    group, depth = hq // hk, chain(lens, hk)
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any() and bool((lse[b] == -math.inf).all())
            continue
        for h in range(hk):
            k, v = (rows_of(c, c[x], b, torch.arange(n))[:, h].double() for x in "kv")
            heads = slice(h * group, (h + 1) * group)
            rows = q[b, heads].double()
            x = d ** -0.5 * rows @ k.T
            size = float((d ** -0.5 * rows.abs() @ k.abs().T).max())
            p, want_lse = torch.softmax(x, dim=-1), torch.logsumexp(x, dim=-1)
            want = p @ v
            tol = out_bound(dtype, d, want, p @ v.abs(), p ** 2 @ v ** 2, size, depth)
            err = (out[b, heads].double() - want).abs()
            assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} times the bound"
            assert bool(((lse[b, heads].double() - want_lse).abs() <= lse_bound(d, want_lse, size, depth)).all())


def _coded(c, what, d):
    """Writes rows that say where they stand: columns[tile or position mod d] = 1."""
    for b, n in enumerate(c["lens"]):
        pos = torch.arange(n, device="cuda")
        row = torch.nn.functional.one_hot(what(pos) % d, d).to(c["k"].dtype)
        yield b, pos, row[:, None].expand(-1, c["k"].shape[2], -1)


@pytest.mark.parametrize("lens", LENS, ids=["one", "several"])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("masked", [False, True], ids=["all", "blocks"])
def test_every_tile_counts_once(kind, lens, masked):
    """Scores of zero: column c of the output is the share of the keys whose tile of 64 is c modulo d, and the sum is their number, both
    of them without rounding before the division."""
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page = kind
    c = make_cache(3, lens, hk, d, page, dtype, fill=0.0)
    c["k"].zero_()
    for b, pos, rows in _coded(c, lambda pos: pos // 64, d):
        c["v"][c["table"][b].long()[pos // page], pos % page] = rows
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    more, on = {}, torch.ones(len(lens), hk, 1 + max(lens) // 48, dtype=torch.bool)
    if masked:
        blocks = -(-c["table"].shape[1] * page // 48)
        on = torch.rand(len(lens), hk, blocks, generator=torch.Generator().manual_seed(5)) < 0.6
        more = dict(block_mask=on.cuda(), k_block_size=48)
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], return_lse=True, **more)
    half = torch.finfo(dtype).eps / 2
    for b, n in enumerate(lens):
        for h in range(hk):
            pos = torch.arange(n)
            pos = pos[on[b, h, pos // 48]]
            count = torch.bincount(pos // 64 % d, minlength=d).double().cuda()
            heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
            if pos.numel() == 0:
                assert not out[b, heads].any() and bool((lse[b, heads] == -math.inf).all())
                continue
            want = count / pos.numel()
            assert bool(((out[b, heads].double() - want).abs() <= want * (half * (1 + half) + 2.0 ** -22)).all())
            exact = math.log(pos.numel())             # the logarithm, its factor and the result: a lost key is 5e-5
            assert float((lse[b, heads].double() - exact).abs().max()) <= (exact + 20) * 2.0 ** -22


@pytest.mark.parametrize("lens", LENS, ids=["one", "several"])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_keys_meet_their_own_values(kind, lens):
    """Query h looks for the keys of the tiles that are h modulo d, and finds their values, as many as there are."""
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page = kind
    c = make_cache(6, lens, hk, d, page, dtype, fill=0.0)
    for b, pos, rows in _coded(c, lambda pos: pos // 64, d):
        at = c["table"][b].long()[pos // page], pos % page
        c["k"][at], c["v"][at] = rows, rows
    for first in range(0, d, hq):
        look = torch.arange(first, first + hq) % d
        q = (60.0 * torch.nn.functional.one_hot(look, d)).to(dtype)[None].repeat(len(lens), 1, 1).cuda()
        out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], 1.0, return_lse=True)
        for b, n in enumerate(lens):
            count = torch.bincount(torch.arange(n) // 64 % d, minlength=d)[look]
            there = count > 0                         # (e^-60 of 20000 others is nothing)
            want = torch.nn.functional.one_hot(look, d).double()
            err = (out[b].cpu().double() - want).abs()[there]
            assert err.numel() == 0 or float(err.max()) <= torch.finfo(dtype).eps / 2 + 2.0 ** -20
            exact = 60.0 + count[there].double().log()
            # a score of 86.6 in the log2 domain, rounded twice, and the sum
            assert bool(((lse[b].cpu().double()[there] - exact).abs() <= 100 * 2.0 ** -22).all())


@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 64, 16), (torch.float32, 64, 16), (torch.float16, 33, 7)])
def test_key_weights_of_other_strides(dtype, d, page):
    """Heads before sequences in memory, and more columns than positions: the weights of a contiguous call, and nothing beside them."""
    import hbsattn_b200 as hb
    lens = [100, 33, 5]
    c = make_cache(7, lens, 2, d, page, dtype)
    q = torch.randn(3, 8, d, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    size = c["table"].shape[1] * page
    want = torch.zeros(3, 2, size, device="cuda")
    hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=want)
    assert len({float(x) for x in want.sum(dim=-1).flatten()}) > 1 and bool((want[:, 0] != want[:, 1]).any())
    memory = torch.zeros(2, 3, size + 3, device="cuda")
    hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=memory.transpose(0, 1))
    assert torch.equal(memory.transpose(0, 1)[:, :, :size], want)
    assert not memory[:, :, size:].any()
    for b, n in enumerate(lens):
        assert not memory[:, b, n:].any()
