"""Attention of one new token over a paged cache against the definition in 64 bits: every kernel, type, layout and split, lengths of
zero, one and around the tile sizes, masks that leave nothing, what must not be looked at, and the states in between (graphs,
streams, bad pages)."""
import math

import pytest
import torch

from cache_helpers import attention_exact, attention_tolerance, make_cache, score_error

pytestmark = pytest.mark.gpu


def _q(seed, batch, nhead_q, d, dtype, factor=2.0):
    return (factor * torch.randn(batch, nhead_q, d, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def _check(q, c, out, lse, **more):
    want, want_lse, spread, weights, size = attention_exact(q, c, **more)
    d, n = q.shape[2], max(c["lens"] + [1])
    tol = attention_tolerance(q.dtype, d, n, want, spread, size)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} times the bound, {float(err.max()):.3g} at most"
    if lse is not None:
        assert torch.equal(lse == -math.inf, want_lse == -math.inf)
        live = want_lse > -math.inf
        # ln of a sum: the scores' error, the sum's, and the rounding of the value itself
        tol = score_error(d, size) + n * 2.0 ** -23 + 2.0 ** -20 + want_lse[live].abs() * 2.0 ** -22
        assert bool(((lse.double() - want_lse)[live].abs() <= tol).all())
    return weights, size


def _weights_check(w, start, weights, d, n, size):
    c32 = 2 * score_error(d, size) + n * 2.0 ** -22 + 2.0 ** -18       # two scores, the sum behind lse, lse in 32 bits and ln 2 twice
    tol = c32 * weights + 2.0 ** -23 * (start.double() + weights) + 1e-30
    err = (w.double() - start.double() - weights).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} times the bound"
    assert torch.equal(w[weights == 0], start[weights == 0])


KINDS = [
    # dtype, nhead_q, nhead_k, d, page, layout
    (torch.bfloat16, 8, 2, 128, 16, "nhd"),
    (torch.bfloat16, 8, 8, 64, 64, "hnd"),
    (torch.float16, 6, 2, 96, 48, "nhd"),
    (torch.float16, 16, 1, 256, 32, "hnd"),
    (torch.bfloat16, 20, 1, 128, 128, "nhd"),      # more than 16 heads of a group: two row tiles
    (torch.bfloat16, 80, 1, 64, 16, "nhd"),        # more than 32: chunks
    (torch.float16, 3, 3, 16, 16, "nhd"),
    (torch.bfloat16, 34, 2, 40, 80, "nhd"),
    (torch.float32, 8, 2, 64, 16, "nhd"),
    (torch.float32, 40, 1, 128, 20, "hnd"),
    (torch.bfloat16, 4, 2, 64, 1, "nhd"),          # page sizes and head dimensions of the CUDA-core kernel
    (torch.float16, 6, 3, 33, 7, "nhd"),
    (torch.float32, 5, 1, 250, 16, "nhd"),
]
IDS = [f"{str(k[0])[6:]}_{k[1]}x{k[2]}_d{k[3]}_p{k[4]}_{k[5]}" for k in KINDS]
LENS = [1, 63, 64, 65, 0, 17, 300, 1029, 16, 128]


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_against_definition(kind):
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page, layout = kind
    c = make_cache(1, LENS, hk, d, page, dtype, layout=layout)
    q = _q(2, len(LENS), hq, d, dtype)
    start = torch.rand(len(LENS), hk, c["table"].shape[1] * page, generator=torch.Generator().manual_seed(3)).cuda()
    w = start.clone()
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w, return_lse=True)
    assert hb.last_status()[0] == 0
    assert out.is_contiguous() and out.dtype == dtype and lse.dtype == torch.float32
    weights, size = _check(q, c, out, lse)
    _weights_check(w, start, weights, d, max(LENS), size)
    again = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
    assert torch.equal(out, again)


@pytest.mark.parametrize("k_block", [16, 48, 64, 80, 128, 400])
@pytest.mark.parametrize("kind", [KINDS[0], KINDS[2], KINDS[4], KINDS[8], KINDS[11]], ids=[IDS[0], IDS[2], IDS[4], IDS[8], IDS[11]])
def test_block_mask(kind, k_block):
    import hbsattn_b200 as hb
    dtype, hq, hk, d, page, layout = kind
    c = make_cache(4, LENS, hk, d, page, dtype, layout=layout)
    q = _q(5, len(LENS), hq, d, dtype)
    size = c["table"].shape[1] * page
    blocks = -(-size // k_block) + 1
    mask = torch.rand(len(LENS), hk, blocks, generator=torch.Generator().manual_seed(6)) < 0.5
    mask[3] = False                                   # nothing left
    mask[6, 0] = False
    mask[7] = False
    mask[7, :, 1029 // k_block] = True                # the last, ragged block alone
    mask = mask.cuda()
    for b in range(len(LENS)):                        # what the mask leaves out is not even looked at
        pos = torch.arange(LENS[b]).cuda()
        for h in range(hk):
            off = pos[~mask[b, h, pos // k_block]]
            for t in (c["k"], c["v"]):
                t[c["table"][b].long()[off // page], off % page, h] = math.nan
    start = torch.zeros(len(LENS), hk, size + 5).cuda()
    w = start.clone()
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], block_mask=mask, k_block_size=k_block, key_weights=w, return_lse=True)
    weights, x = _check(q, c, out, lse, mask=mask, k_block=k_block)
    _weights_check(w[..., :size], start[..., :size], weights, d, max(LENS), x)
    assert not out[3].any() and bool((lse[3] == -math.inf).all())
    strided = torch.zeros(hk, len(LENS), 2 * blocks, dtype=torch.bool, device="cuda")[:, :, ::2].transpose(0, 1)
    strided.copy_(mask)
    assert torch.equal(out, hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], block_mask=strided, k_block_size=k_block))


@pytest.mark.parametrize("dtype,hq,hk,d", [(torch.bfloat16, 4, 1, 128), (torch.float16, 8, 1, 64), (torch.float32, 2, 1, 64), (torch.bfloat16, 40, 1, 256)])
@pytest.mark.parametrize("lens", [[20000], [9000, 1, 0, 12000], [0, 0]])
def test_long_rows_are_split_and_joined(dtype, hq, hk, d, lens):
    import hbsattn_b200 as hb
    c = make_cache(7, lens, hk, d, 64, dtype, fill=0.0)
    q = _q(8, len(lens), hq, d, dtype)
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], return_lse=True)
    _check(q, c, out, lse)
    for _ in range(3):
        assert torch.equal(out, hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"]))


@pytest.mark.parametrize("dtype,hq,hk,d,page", [(torch.bfloat16, 16, 4, 64, 64), (torch.float16, 8, 4, 128, 16), (torch.bfloat16, 16, 4, 256, 64), (torch.bfloat16, 36, 2, 128, 32),
                                               (torch.float16, 40, 2, 256, 16)])
def test_many_rounds_of_the_ring(dtype, hq, hk, d, page):
    """Every CTA goes through its stages dozens of times, over several rows."""
    import hbsattn_b200 as hb
    lens = [20000, 15001, 9000, 20011, 64, 17000, 12345, 19999]
    c = make_cache(70, lens, hk, d, page, dtype, fill=0.0)
    q = _q(71, len(lens), hq, d, dtype)
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], return_lse=True)
    _check(q, c, out, lse)


@pytest.mark.parametrize("batch,n,hq,hk,d", [(300, 40, 8, 2, 64), (1500, 5, 1, 1, 32), (64, 700, 16, 8, 128)])
def test_many_sequences(batch, n, hq, hk, d):
    import hbsattn_b200 as hb
    lens = [(7 * i) % n for i in range(batch)]
    c = make_cache(9, lens, hk, d, 16, torch.bfloat16)
    q = _q(10, batch, hq, d, torch.bfloat16)
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], return_lse=True)
    _check(q, c, out, lse)


@pytest.mark.parametrize("family", ["sm100", "generic"])
def test_sharp_and_flat_scores_and_scales(family):
    import hbsattn_b200 as hb
    lens = [700, 65]
    c = make_cache(11, lens, 2, 64, 16, torch.float16)
    hb.set_kernel_family(family)
    try:
        for factor, scale in ((30.0, None), (0.0, None), (1.0, 0.7), (1.0, 1e-3)):
            q = _q(12, 2, 8, 64, torch.float16, factor)
            out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], scale, return_lse=True)
            _check(q, c, out, lse, scale=scale)
    finally:
        hb.set_kernel_family("auto")
    q = _q(12, 2, 8, 64, torch.float16, 1.0)
    for scale in (-0.5, 0.0):                         # the CUDA-core kernel takes these
        out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], scale, return_lse=True)
        _check(q, c, out, lse, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities(dtype):
    """A key whose score is -inf has no weight; a row of nothing but such keys sees none."""
    import hbsattn_b200 as hb
    c = make_cache(13, [90, 40], 1, 64, 16, dtype)
    q = torch.ones(2, 2, 64, dtype=dtype, device="cuda")
    table = c["table"].long()
    for pos in (0, 33, 89):
        c["k"][table[0, pos // 16], pos % 16] = -math.inf
    for pos in range(40):
        c["k"][table[1, pos // 16], pos % 16] = -math.inf
    w = torch.zeros(2, 1, c["table"].shape[1] * 16, device="cuda")
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w, return_lse=True)
    seen = [p for p in range(90) if p not in (0, 33, 89)]
    at = torch.tensor(seen, device="cuda")
    k, v = (t[table[0, at // 16], at % 16, 0].double() for t in (c["k"], c["v"]))
    p = torch.softmax(q[0].double() @ k.T / 8, dim=-1)
    size = float(k.abs().sum(dim=-1).max()) / 8
    tol = attention_tolerance(dtype, 64, 90, p @ v, p @ v.abs(), size)
    assert bool(((out[0].double() - p @ v).abs() <= tol).all())
    assert not w[0, 0, [0, 33, 89]].any() and bool((w[0, 0, seen] > 0).all())
    assert not out[1].any() and bool((lse[1] == -math.inf).all()) and not w[1].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("masked", [False, True])
def test_lengths_and_pages_out_of_range(dtype, masked):
    """Lengths are cut to the cache, positions on pages that do not exist take part in nothing, and the status says so."""
    import hbsattn_b200 as hb
    c = make_cache(14, [64, 64, 64, 64], 2, 64, 16, dtype, extra_pages=0)
    q = _q(15, 4, 4, 64, dtype)
    mask = torch.ones(4, 2, 4, dtype=torch.bool, device="cuda") if masked else None
    more = dict(block_mask=mask, k_block_size=16) if masked else {}
    out = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], **more)
    assert hb.last_status()[:2] == [0, 0]
    lens = torch.tensor([64, 1000, -3, 64], dtype=torch.int32, device="cuda")
    got, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], lens, return_lse=True, **more)
    assert hb.last_status()[0] == 3
    assert torch.equal(got[[0, 1, 3]], out[[0, 1, 3]]) and not got[2].any() and bool((lse[2] == -math.inf).all())
    for bad in (-1, c["k"].shape[0], 2 ** 31 - 1):
        table = c["table"].clone()
        table[3, 1] = bad
        w = torch.zeros(4, 2, 64, device="cuda")
        got = hb.paged_attention(q, c["k"], c["v"], table, c["cache_lens"], key_weights=w, **more)
        assert hb.last_status()[:2] == [3, 3]
        assert torch.equal(got[:3], out[:3])
        assert not w[3, :, 16:32].any() and bool((w[3, :, :16] > 0).all()) and bool((w[3, :, 32:] > 0).all())
        leaves = torch.ones(4, 2, 4, dtype=torch.bool, device="cuda")
        leaves[3, :, 1] = False
        want, _, spread, _, size = attention_exact(q, c, mask=leaves, k_block=16)
        assert bool(((got.double() - want).abs() <= attention_tolerance(dtype, 64, 64, want, spread, size)).all())


def test_shared_pages_and_offsets_beyond_32_bits():
    import hbsattn_b200 as hb
    pages = (2 ** 31 // (64 * 8 * 64)) + 40
    k, v = (torch.zeros(pages, 64, 8, 64, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    g = torch.Generator(device="cuda").manual_seed(16)
    for t in (k, v):
        t[-40:] = torch.randn(40, 64, 8, 64, generator=g, device="cuda", dtype=torch.bfloat16)
    table = torch.arange(pages - 40, pages, dtype=torch.int32, device="cuda")[None].expand(3, 40)    # three sequences, one set of pages
    lens = [2500, 640, 1]
    c = dict(k=k, v=v, table=table, page=64, lens=lens, cache_lens=torch.tensor(lens, device="cuda"))   # int64 lengths
    q = _q(17, 3, 16, 64, torch.bfloat16)
    out, lse = hb.paged_attention(q, k, v, table, c["cache_lens"], return_lse=True)
    _check(q, c, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_inputs(dtype):
    import hbsattn_b200 as hb
    c = make_cache(18, [100, 33, 5], 2, 64, 16, dtype)
    q = _q(19, 3, 8, 64, dtype)
    want = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
    kv = torch.stack([c["k"], c["v"]], dim=1)                                        # one tensor for both
    assert torch.equal(want, hb.paged_attention(q, kv[:, 0], kv[:, 1], c["table"], c["cache_lens"]))
    wide = torch.zeros(*c["k"].shape[:3], 130, dtype=dtype, device="cuda")[..., 1:65]   # rows that are not aligned
    wide.copy_(c["k"])
    got = hb.paged_attention(q, wide, c["v"], c["table"], c["cache_lens"])
    _check(q, c, got, None)
    apart = torch.zeros(8, 3, 128, dtype=dtype, device="cuda")[..., ::2].transpose(0, 1)
    apart.copy_(q)
    _check(q, c, hb.paged_attention(apart, c["k"], c["v"], c["table"], c["cache_lens"]), None)
    table = torch.zeros(c["table"].shape[1], 3, dtype=torch.int32, device="cuda").t()
    table.copy_(c["table"])
    assert torch.equal(want, hb.paged_attention(q, c["k"], c["v"], table, c["cache_lens"]))
    w = torch.zeros(2, 3, c["table"].shape[1] * 16 + 3, device="cuda")
    hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w.transpose(0, 1))
    assert bool(((w.transpose(0, 1)[:, :, :5].sum(dim=-1) > 0)).all())


def test_two_graphs_and_a_side_stream():
    """Captured calls own their workspace: two of them replayed in turn and at once, and an eager call on another stream between."""
    import hbsattn_b200 as hb
    sets = []
    for i, lens in enumerate(([3000, 17, 800], [1, 5000, 64])):
        c = make_cache(20 + i, lens, 2, 128, 64, torch.bfloat16)
        q = _q(30 + i, 3, 8, 128, torch.bfloat16)
        hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
        sets.append((c, q, graph, out))
    streams = [torch.cuda.Stream() for _ in sets]
    for round_ in range(3):
        for (c, q, graph, out), s in zip(sets, streams):
            q.copy_(_q(40 + round_, 3, 8, 128, torch.bfloat16))
            out.zero_()
            c["cache_lens"].copy_(torch.tensor([n - round_ if n > round_ else 0 for n in c["lens"]], dtype=torch.int32))
        torch.cuda.synchronize()
        for (c, q, graph, out), s in zip(sets, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for c, q, graph, out in sets:
            assert torch.equal(out, hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"]))
            want, _, spread, _, size = attention_exact(q, c, lens=c["cache_lens"].tolist())
            assert bool(((out.double() - want).abs() <= attention_tolerance(q.dtype, 128, 5000, want, spread, size)).all())


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_a_call_that_gives_up_returns_nan(dtype, d):
    """The tensor-core kernel's loader stays silent, every other wait runs out with nothing in flight."""
    import hbsattn_b200 as hb
    from hbsattn_b200 import _lib
    lib = _lib.load()
    c = make_cache(50, [700, 3, 0], 2, d, 16, dtype)
    q = _q(51, 3, 8, d, dtype)
    w = torch.zeros(3, 2, c["table"].shape[1] * 16, device="cuda")
    before = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"])
    try:
        lib.hbsa_debug_set_wait_budget(2_000_000, 1)
        out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w, return_lse=True)
        assert hb.last_status()[0] == _lib.HBSA_STATUS_WAIT_LIMIT
        assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all()) and not w.any()
    finally:
        lib.hbsa_debug_set_wait_budget(0, 0)
    assert torch.equal(before, hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"]))
    assert hb.last_status()[0] == 0


def test_refusals():
    import hbsattn_b200 as hb
    c = make_cache(60, [40, 3], 2, 64, 16, torch.bfloat16)
    q = _q(61, 2, 4, 64, torch.bfloat16)
    w = torch.zeros(2, 2, c["table"].shape[1] * 16, device="cuda")
    mask = torch.ones(2, 2, c["table"].shape[1], dtype=torch.bool, device="cuda")

    def call(q=q, k=c["k"], v=c["v"], table=c["table"], lens=c["cache_lens"], **more):
        return hb.paged_attention(q, k, v, table, lens, **more)
    call(key_weights=w, block_mask=mask, k_block_size=16)
    bad = [dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q.half()), dict(q=q[:, :3]), dict(v=c["v"][:-1]), dict(k=c["k"].half()), dict(lens=c["cache_lens"][:1]),
           dict(table=c["table"][0]), dict(lens=c["cache_lens"].float()), dict(key_weights=w[..., :-1]), dict(key_weights=w.double()),
           dict(key_weights=w[:1].expand(2, -1, -1)), dict(block_mask=mask), dict(block_mask=mask, k_block_size=24),
           dict(block_mask=mask[..., :-1], k_block_size=16), dict(block_mask=mask.int(), k_block_size=16), dict(block_mask=mask[:, :1], k_block_size=16)]
    for more in bad:
        with pytest.raises(AssertionError):
            call(**more)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(q=q.cpu())
    for name, t in (("q", q), ("k", c["k"]), ("v", c["v"])):
        with pytest.raises(RuntimeError, match="derivative"):
            call(**{name: t.clone().requires_grad_(True)})
        with torch.no_grad():
            call(**{name: t.clone().requires_grad_(True)})
    hb.set_kernel_family("sm100")
    try:
        with pytest.raises(RuntimeError, match="tensor-core"):
            call(softmax_scale=-1.0)
    finally:
        hb.set_kernel_family("auto")
    empty = hb.paged_attention(q[:0], c["k"], c["v"], c["table"][:0], c["cache_lens"][:0], return_lse=True)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 4)
