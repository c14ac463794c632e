"""The attention weight that a block-sparse prompt gives to its keys, against the definition in 64 bits: both kernel families, types, block
sizes, GQA groups, causal alignment with unequal lengths, rows without keys, and what must not leak in."""
import math

import pytest
import torch

from cache_helpers import score_error
from helpers import make_problem

pytestmark = pytest.mark.gpu


def exact(pr, q, k, lse, scale=None):
    """Weights, and the largest sum of |q_i k_i| of a score."""
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    group, scale = hq // hk, d ** -0.5 if scale is None else scale
    w = torch.zeros(k.shape[0], hk, dtype=torch.float64, device=k.device)
    size, qb, kb = 0.0, 0, 0
    cq, ck = pr["cu_q_list"], pr["cu_k_list"]
    for b in range(len(cq) - 1):
        m, n = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        i, j = torch.arange(m, device=k.device)[:, None], torch.arange(n, device=k.device)[None]
        for h in range(hq if m and n else 0):
            x = scale * q[cq[b]:cq[b + 1], h].double() @ k[ck[b]:ck[b + 1], h // group].double().T
            on = pr["mask"][h // group][qb + i // pr["qbs"], kb + j // pr["kbs"]]
            if pr["causal"]:
                on = on & (i + n - m >= j)
            row = lse[cq[b]:cq[b + 1], h, None].double()
            on = on & (row > -math.inf)
            if bool(on.any()):
                size = max(size, float((abs(scale) * q[cq[b]:cq[b + 1], h].double().abs() @ k[ck[b]:ck[b + 1], h // group].double().abs().T)[on].max()))
            w[ck[b]:ck[b + 1], h // group] += torch.where(on, torch.exp(x - torch.where(row > -math.inf, row, 0.0)), 0.0).sum(dim=0)
        qb, kb = qb - (-m // pr["qbs"]), kb - (-n // pr["kbs"])
    return w, size


def check(pr, w, want, size, lse, d, group):
    # relative: the score's error and its rounding with the lse in the log2 domain, the exponential (2^-21), sums of fp32 terms
    top = float(lse[lse.abs() < math.inf].abs().max()) if bool((lse.abs() < math.inf).any()) else 0.0
    rows = max([b - a for a, b in zip(pr["cu_q_list"], pr["cu_q_list"][1:])]) * group
    c = 2 * score_error(d, size) + (top + size) * 2.0 ** -22 + rows * 2.0 ** -24 + 2.0 ** -20
    err = (w.double() - want).abs()
    assert w.dtype == torch.float32 and w.shape == want.shape
    assert bool((err <= c * want).all()), f"off by {float((err / (c * want).clamp(min=1e-300)).max()):.2f} times the bound"


CASES = [
    # hq, hk, d, qbs, kbs, causal, dtype
    (2, 2, 128, 128, 128, True, torch.bfloat16),
    (8, 2, 64, 80, 48, False, torch.float16),
    (3, 1, 96, 48, 144, True, torch.bfloat16),
    (8, 1, 32, 16, 16, True, torch.float16),
    (32, 1, 64, 16, 80, True, torch.bfloat16),
    (12, 2, 128, 64, 256, False, torch.float16),
    (4, 2, 256, 128, 64, True, torch.bfloat16),
    (64, 1, 136, 32, 272, False, torch.float16),
    (4, 2, 64, 64, 64, True, torch.float32),
    (3, 3, 200, 48, 80, False, torch.float32),
    (6, 2, 30, 32, 16, True, torch.bfloat16),
]


@pytest.mark.parametrize("lens", [([203, 150, 77], [203, 150, 77]), ([1, 130, 64, 33], [300, 129, 1, 33]), ([400], [150])], ids=["equal", "unequal", "more_rows"])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}x{c[1]}_d{c[2]}_{c[3]}x{c[4]}_{str(c[6])[6:]}" for c in CASES])
def test_against_definition(case, lens):
    import hbsattn_b200 as hb
    hq, hk, d, qbs, kbs, causal, dtype = case
    pr = make_problem(81, *lens, hq, hk, d, qbs, kbs, causal, dtype, 0.6, None)
    q = 2 * pr["q"]
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], qbs, kbs, causal)
    _, lse = hb.HBSAttention_with_lse(q, pr["k"], pr["v"], *rest)
    w = hb.attention_key_weights(q, pr["k"], lse, *rest)
    assert hb.last_status()[0] == 0
    want, size = exact(pr, q, pr["k"], lse)
    check(pr, w, want, size, lse, d, hq // hk)
    assert torch.equal(w, hb.attention_key_weights(q, pr["k"], lse, *rest))
    if dtype != torch.float32 and d % 8 == 0:         # both families take these
        hb.set_kernel_family("generic")
        try:
            check(pr, hb.attention_key_weights(q, pr["k"], lse, *rest), want, size, lse, d, hq // hk)
        finally:
            hb.set_kernel_family("auto")
    from hbsattn_b200.shard import csr_of_mask
    from oracle import oracle_block_decisions
    inside = torch.from_numpy(oracle_block_decisions(pr["cu_q_list"], pr["cu_k_list"], torch.ones_like(pr["mask"]), qbs, kbs, False)).cuda()
    ptr, idx = csr_of_mask(pr["mask"] & inside)
    if idx.numel():
        got = hb.attention_key_weights_csr(q, pr["k"], lse, pr["cu_q"], pr["cu_k"], ptr, idx, *pr["mask"].shape[1:], qbs, kbs, causal)
        assert torch.equal(w, got)


@pytest.mark.parametrize("hq,hk,d,n", [(8, 8, 128, 4000), (16, 2, 64, 3001), (1, 1, 128, 9000)])
def test_longer_prompts(hq, hk, d, n):
    import hbsattn_b200 as hb
    pr = make_problem(82, [n, 100], [n, 100], hq, hk, d, 128, 128, True, torch.bfloat16, 0.3, "diag")
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], 128, 128, True)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], *rest)
    w = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
    want, size = exact(pr, pr["q"], pr["k"], lse)
    check(pr, w, want, size, lse, d, hq // hk)
    # every row's weights sum to one
    assert abs(float(w.double().sum()) / (hq * (n + 100)) - 1) < 1e-5


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("case", [CASES[0], CASES[1], CASES[4], CASES[6], CASES[8]], ids=["d128", "d64", "mqa", "d256", "fp32"])
def test_isolation(case, value):
    """Rows of another sample, behind the last one, and rows that see no key: whatever they hold, other samples' weights keep their bits."""
    import hbsattn_b200 as hb
    hq, hk, d, qbs, kbs, causal, dtype = case
    pr = make_problem(83, [203, 150, 77], [203, 150, 77], hq, hk, d, qbs, kbs, causal, dtype, 0.6, "diag" if causal else "first")
    q, k, v = (torch.cat([pr[n], torch.zeros(70, *pr[n].shape[1:], dtype=dtype, device="cuda")]) for n in "qkv")
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], qbs, kbs, causal)
    _, lse = hb.HBSAttention_with_lse(q, k, v, *rest)
    clean = hb.attention_key_weights(q, k, lse, *rest)
    assert not clean[430:].any()
    for rows in (slice(203, 353), slice(430, 500)):
        for which in range(2):
            t = [q.clone(), k.clone()]
            t[which][rows] = value
            got = hb.attention_key_weights(*t, lse, *rest)
            assert torch.equal(got[:203], clean[:203]) and torch.equal(got[353:430], clean[353:430]) and not got[430:].any()
    dead = lse.clone()
    dead[10:40] = -math.inf
    without = hb.attention_key_weights(q, k, dead, *rest)
    bad = q.clone()
    bad[10:40] = value
    assert torch.equal(without, hb.attention_key_weights(bad, k, dead, *rest))


def test_more_rows_than_keys_and_strided_inputs():
    import hbsattn_b200 as hb
    pr = make_problem(84, [230], [100], 4, 2, 128, 64, 64, True, torch.bfloat16, 1.0, None)
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], 64, 64, True)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], *rest)
    w = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
    bad = pr["q"].clone()
    bad[:130] = math.nan                              # these rows see no key
    assert torch.equal(w, hb.attention_key_weights(bad, pr["k"], lse, *rest))
    turned = lse.t().contiguous().t()
    qk = torch.cat([pr["q"], torch.zeros_like(pr["q"])], dim=2)[..., :128]
    heads_first = pr["k"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(w, hb.attention_key_weights(qk, heads_first, turned, *rest))
    odd = torch.zeros(*pr["k"].shape[:2], 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(pr["k"])
    want, size = exact(pr, pr["q"], pr["k"], lse)
    check(pr, hb.attention_key_weights(pr["q"], odd, lse, *rest), want, size, lse, 128, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_mask_that_contradicts_the_lengths(dtype):
    import hbsattn_b200 as hb
    pr = make_problem(85, [100, 60], [100, 60], 2, 1, 64, 64, 64, True, dtype, 0.7, "diag")
    lse = torch.zeros(160, 2, device="cuda")
    w = hb.attention_key_weights(pr["q"], pr["k"], lse, pr["cu_q"], pr["cu_k"], pr["mask"][:, :, :-1], 64, 64, True)
    assert hb.last_status()[0] == 1 and not w.any()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_a_call_that_gives_up_returns_nan(dtype, d):
    import hbsattn_b200 as hb
    from hbsattn_b200 import _lib
    lib = _lib.load()
    pr = make_problem(86, [256, 384], [256, 384], 4, 2, d, 128, 128, True, dtype, 0.6, "diag")
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], 128, 128, True)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], *rest)
    before = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
    try:
        lib.hbsa_debug_set_wait_budget(2_000_000, 1)
        w = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
        assert hb.last_status()[0] == _lib.HBSA_STATUS_WAIT_LIMIT and bool(torch.isnan(w).all())
    finally:
        lib.hbsa_debug_set_wait_budget(0, 0)
    assert torch.equal(before, hb.attention_key_weights(pr["q"], pr["k"], lse, *rest))
    assert hb.last_status()[0] == 0


def test_refusals_and_empty_inputs():
    import hbsattn_b200 as hb
    pr = make_problem(87, [100, 60], [100, 60], 2, 1, 64, 64, 64, True, torch.bfloat16, 0.7, "diag")
    lse = torch.zeros(160, 2, device="cuda")

    def call(q=pr["q"], k=pr["k"], lse=lse, mask=pr["mask"], qbs=64, cu=pr["cu_q"]):
        return hb.attention_key_weights(q, k, lse, cu, pr["cu_k"], mask, qbs, 64, True)
    call()
    for more in (dict(lse=lse.half()), dict(lse=lse[:-1]), dict(mask=pr["mask"].int()), dict(mask=pr["mask"][0]), dict(qbs=24), dict(k=pr["k"].half()),
                 dict(q=pr["q"][..., :32]), dict(cu=pr["cu_q"][:-1])):
        with pytest.raises(AssertionError):
            call(**more)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(lse=lse.cpu())
    with pytest.raises(RuntimeError, match="derivative"):
        call(q=pr["q"].clone().requires_grad_(True))
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    w = hb.attention_key_weights(pr["q"][:0], pr["k"], lse[:0], none, pr["cu_k"], pr["mask"], 64, 64, True)
    assert w.shape == (160, 1) and not w.any()
