"""fp16 decoding beside keys that outweigh the others by far (attention sinks): probabilities of 2^-24 to 2^-28 of the largest are still
counted, one by one rounded by no more than half a step of fp16."""
import math

import pytest
import torch

from cache_helpers import score_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nats", [9.0, 17.0, 18.0, 19.0])
@pytest.mark.parametrize("nhead_q,d", [(1, 64), (20, 64), (4, 128), (20, 128), (8, 256)])
def test_many_small_terms_beside_sinks(nhead_q, d, nats):
    import hbsattn_b200 as hb
    # Every warp that works on the start of a row meets a sink: one key in sixteen of the first 512.  Sinks have a value of zero, so the output is
    # the share of the other keys, 2048 n e^-nats / (32 + n e^-nats).  160 sequences on the same pages: most rows are one CTA's alone.
    batch, n, page = 160, 8192, 64
    sinks = torch.arange(0, 512, 16)
    k = torch.zeros(n, d)
    k[sinks, 0] = nats
    v = torch.full((n, d), 2048.0)
    v[sinks] = 0.0
    k, v = (t.to(torch.float16).reshape(n // page, page, 1, d).cuda() for t in (k, v))
    q = torch.zeros(batch, nhead_q, d, dtype=torch.float16)
    q[..., 0] = 1.0
    table = torch.arange(n // page, dtype=torch.int32)[None].repeat(batch, 1).cuda()
    lens = torch.full((batch,), n, dtype=torch.int32).cuda()
    out, lse = hb.paged_attention(q.cuda(), k, v, table, lens, 1.0, return_lse=True)
    rest = (n - len(sinks)) * math.exp(-nats)
    want = 2048.0 * rest / (len(sinks) + rest)
    # half a step of fp16 for P, the same for all of them, and half a step for the output; scores in 32 bits, twice (P and sum); sums of at most
    # 512 terms a lane one after the other, eight warps and two parts; exponentials, logarithms and the division
    half = 2.0 ** -11
    c32 = 2 * score_error(d, nats) + 522 * 2.0 ** -23 + 2.0 ** -20
    assert want * half > 2.0 ** -25                       # the output is a normal number
    err = (out.double() - want).abs().max()
    assert float(err) <= want * (2 * half * (1 + half) + c32), f"off by {float(err) / want:.3g} of the value"
    exact = nats + math.log(len(sinks) + rest)
    assert float((lse.double() - exact).abs().max()) <= score_error(d, nats) + 522 * 2.0 ** -23 + 2.0 ** -20 + exact * 2.0 ** -22


@pytest.mark.parametrize("scale", [2.0 ** e for e in range(-4, 12)] + [3.0, 100.0])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_equal_scores_of_any_size(d, scale):
    """Scores up to 2^40: all equal, so every key has the same weight, whatever is subtracted before the exponential; one key more far below."""
    import hbsattn_b200 as hb
    lens, page = [1, 100, 700, 0], 16
    g = torch.Generator().manual_seed(1)
    pages = 45
    k = torch.full((pages, page, 1, d), 2.0 ** 12).to(torch.float16).cuda()
    v = torch.randn(pages, page, 1, d, generator=g).to(torch.float16).cuda()
    k[0, 0] = -1.0
    table = torch.arange(pages, dtype=torch.int32)[None].repeat(len(lens), 1).cuda()
    q = torch.full((len(lens), 6, d), 2.0 ** 11).to(torch.float16)
    q[:, 1] *= -1.0                                        # the sum's sign
    q = q.cuda()
    out = hb.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32).cuda(), scale)
    rows = v.reshape(-1, d).double()
    half = 2.0 ** -11
    for b, n in enumerate(lens):
        for h in range(6):
            low = h == 1                                   # the first key alone has the largest score there
            some = rows[:1] if low or n == 1 else rows[1:n]
            want = some.mean(dim=0) if n > 0 else torch.zeros(d, dtype=torch.float64, device="cuda")
            spread = some.abs().mean(dim=0) if n > 0 else want
            tol = half * want.abs() + (half + 700 * 2.0 ** -23 + 2.0 ** -20) * spread * (1 + half) + 2.0 ** -25
            assert bool(((out[b, h].double() - want).abs() <= tol).all()), (n, h)
