"""Groups of up to 8 heads in 16 bits: the probabilities lose nothing, so the output is off by its own rounding and what 32 bits leave; infinite values
come through as they do with one product."""
import math

import pytest
import torch

from cache_helpers import make_cache, rows_of, score_error
from paged_bounds import chain

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, 8, 1, 64, 64), (torch.float16, 16, 2, 64, 16), (torch.bfloat16, 8, 2, 128, 64), (torch.float16, 7, 1, 96, 48), (torch.bfloat16, 3, 3, 256, 32),
         (torch.float16, 8, 1, 256, 16), (torch.bfloat16, 40, 8, 16, 16), (torch.float16, 8, 8, 136, 80)]
IDS = [f"{str(k[0])[6:]}_{k[1]}x{k[2]}_d{k[3]}_p{k[4]}" for k in KINDS]


@pytest.mark.parametrize("masked", [False, True], ids=["all", "blocks"])
@pytest.mark.parametrize("factor", [0.3, 3.0])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_nothing_but_the_outputs_rounding(kind, factor, masked):
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page = kind
    lens = [1, 17, 300, 2029, 0, 9001]
    c = make_cache(1, lens, hk, d, page, dtype)
    q = (factor * torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(2))).to(dtype).cuda()
    on, more = None, {}
    if masked:
        on = torch.rand(len(lens), hk, -(-c["table"].shape[1] * page // 64), generator=torch.Generator().manual_seed(3)).cuda() < 0.7
        more = dict(block_mask=on, k_block_size=64)
    out = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], **more)
    group, half, depth = hq // hk, torch.finfo(dtype).eps / 2, chain(lens, hk)
    for b, n in enumerate(lens):
        for h in range(hk):
            pos = torch.arange(n, device="cuda")
            if masked:
                pos = pos[on[b, h, pos // 64]]
            heads = slice(h * group, (h + 1) * group)
            if pos.numel() == 0:
                assert not out[b, heads].any()
                continue
            k, v = (rows_of(c, c[x], b, pos)[:, h].double() for x in "kv")
            rows = q[b, heads].double()
            x = d ** -0.5 * rows @ k.T
            size = float((d ** -0.5 * rows.abs() @ k.abs().T).max())
            p = torch.softmax(x, dim=-1)
            want, spread = p @ v, p @ v.abs()
            # the output's rounding; what two terms leave of p (half a step of half a step; fp16: 2^-39 of the largest p at least); scores in p and in
            # the sum, sums, exponentials and the division in 32 bits
            c32 = 2 * score_error(d, size) + 2 * depth * 2.0 ** -24 + 2.0 ** -20
            tol = half * want.abs() * (1 + 2 * half) + (half * half + c32) * spread + 2.0 ** -25
            if dtype == torch.float16:
                tol = tol + 2.0 ** -39 * v.abs().sum(dim=0)
            err = (out[b, heads].double() - want).abs()
            assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} times the bound"


@pytest.mark.parametrize("kind", KINDS + [(torch.bfloat16, 16, 1, 64, 16)], ids=IDS + ["bfloat16_16x1_d64_p16"])
def test_infinite_values(kind):
    """An infinite value of a key with weight makes its column infinite, two of both signs make it NaN, and the other columns know nothing of it."""
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page = kind
    lens = [300, 64, 1]
    c = make_cache(4, lens, hk, d, page, dtype)
    q = (0.5 * torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(5))).to(dtype).cuda()
    clean = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
    for b, n in enumerate(lens):
        for col, values in ((0, {n // 2: math.inf}), (3, {0: -math.inf}), (5, {n - 1: math.inf, n // 3: math.inf}), (7, {0: math.inf, n - 1: -math.inf})):
            for pos, x in values.items():
                c["v"][int(c["table"][b, pos // page]), pos % page, :, col] = x
    out = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
    for b, n in enumerate(lens):
        assert bool((out[b, :, 0] == math.inf).all()) and bool((out[b, :, 3] == -math.inf).all()) and bool((out[b, :, 5] == math.inf).all())
        assert bool(torch.isnan(out[b, :, 7]).all() if n > 1 else (out[b, :, 7] == -math.inf).all())
    rest = [i for i in range(d) if i not in (0, 3, 5, 7)]
    assert torch.equal(out[..., rest], clean[..., rest])
