"""Writing into a paged cache, choosing what stays, and moving it: exact copies and exact choices, compared element by element, pages
that belong to nobody included."""
import math

import pytest
import torch

from cache_helpers import make_cache

pytestmark = pytest.mark.gpu

KINDS = [
    # dtype, nhead_k, d, page, layout
    (torch.bfloat16, 2, 128, 16, "nhd"),
    (torch.float16, 8, 64, 64, "hnd"),
    (torch.float32, 3, 96, 48, "nhd"),
    (torch.bfloat16, 1, 33, 7, "nhd"),
    (torch.float32, 2, 250, 1, "hnd"),
    (torch.float16, 5, 8, 256, "nhd"),
]
IDS = [f"{str(k[0])[6:]}_{k[1]}_d{k[2]}_p{k[3]}_{k[4]}" for k in KINDS]


def same(a, b):
    """Bit for bit, NaN included."""
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _at(c, b, positions):
    positions = torch.as_tensor(positions, device=c["table"].device)
    return c["table"][b].long()[positions // c["page"]], positions % c["page"]


# ------------------------------------------------------------------------------------------------------------------ append
def _appended(c, k, v, cu):
    want = [c["k"].clone(), c["v"].clone()]
    for b in range(len(c["lens"])):
        at = _at(c, b, torch.arange(c["lens"][b], c["lens"][b] + cu[b + 1] - cu[b]))
        for cache, new in zip(want, (k, v)):
            cache[at] = new[cu[b]:cu[b + 1]]
    return want


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [300, 0, 17, 1, 129]], ids=["one", "none", "ragged"])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_append(kind, new):
    import hbsattn_b200 as hb
    dtype, hk, d, page, layout = kind
    c = make_cache(1, [0, 63, 64, 65, 200], hk, d, page, dtype, layout=layout, room=max(new))
    front, behind = 3, 5                              # rows of k and v that belong to no sequence
    cu = [front]
    for n in new:
        cu.append(cu[-1] + n)
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(cu[-1] + behind, hk, d, generator=g, device="cuda").to(dtype) for _ in "kv")
    want = _appended(c, k, v, cu)
    lens = hb.append_to_cache(k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), c["k"], c["v"], c["table"], c["cache_lens"])
    assert hb.last_status()[0] == 0
    assert lens.tolist() == [a + n for a, n in zip(c["lens"], new)] and lens.dtype == torch.int32
    assert same(c["k"], want[0]) and same(c["v"], want[1])
    assert c["cache_lens"].tolist() == c["lens"]


def test_append_many_sequences_and_strided_rows():
    import hbsattn_b200 as hb
    lens = [(13 * i) % 50 for i in range(700)]
    c = make_cache(3, lens, 2, 64, 16, torch.bfloat16, room=1)
    kv = torch.randn(700, 2, 2, 64, device="cuda").to(torch.bfloat16)               # k and v side by side
    k, v = kv[:, 0], kv[:, 1]
    cu = torch.arange(701, device="cuda")                                            # int64
    want = _appended(c, k, v, list(range(701)))
    got = hb.append_to_cache(k, v, cu, c["k"], c["v"], c["table"], c["cache_lens"])
    assert got.tolist() == [n + 1 for n in lens] and same(c["k"], want[0]) and same(c["v"], want[1])
    turned = torch.randn(64, 700, 2, device="cuda").to(torch.bfloat16).permute(1, 2, 0)
    want = _appended(c, turned, v, list(range(701)))
    hb.append_to_cache(turned, v, cu, c["k"], c["v"], c["table"], c["cache_lens"])
    assert same(c["k"], want[0]) and same(c["v"], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_beyond_the_cache(dtype):
    """What has no room or no page is not written, the rest is; lengths are cut to the cache."""
    import hbsattn_b200 as hb
    c = make_cache(4, [40, 40, 40, 40], 2, 64, 16, dtype, extra_pages=0, room=24)     # 64 positions each
    table = c["table"].clone()
    table[2, 3] = c["k"].shape[0]
    table[3, 2] = -1
    new = [30, 3, 20, 24]
    cu = [0, 30, 33, 53, 77]
    k, v = (torch.randn(77, 2, 64, device="cuda").to(dtype) for _ in "kv")
    want = [c["k"].clone(), c["v"].clone()]
    for b, n in enumerate(new):
        for i in range(n):
            pos = 40 + i
            if pos >= 64 or (b == 2 and pos >= 48) or (b == 3 and 32 <= pos < 48):
                continue
            for cache, t in zip(want, (k, v)):
                cache[int(c["table"][b, pos // 16]), pos % 16] = t[cu[b] + i]
    lens = hb.append_to_cache(k, v, torch.tensor(cu, device="cuda"), c["k"], c["v"], table, c["cache_lens"])
    assert hb.last_status()[:2] == [3, 0]
    assert lens.tolist() == [64, 43, 60, 64] and same(c["k"], want[0]) and same(c["v"], want[1])


def test_append_refusals():
    import hbsattn_b200 as hb
    c = make_cache(5, [4, 3], 2, 64, 16, torch.bfloat16, room=1)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")

    def call(k=k, v=k, cu=cu, kc=c["k"], vc=c["v"], table=c["table"], lens=c["cache_lens"]):
        return hb.append_to_cache(k, v, cu, kc, vc, table, lens)
    call()
    for more in (dict(k=k[:1]), dict(k=k[..., :32], v=k[..., :32]), dict(k=k.half(), v=k.half()), dict(cu=cu[:-1]), dict(kc=c["k"][:1].expand(8, -1, -1, -1), vc=c["v"][:1].expand(8, -1, -1, -1)),
                 dict(kc=c["k"][..., 0]), dict(lens=c["cache_lens"][:1])):
        with pytest.raises(AssertionError):
            call(**more)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(cu=cu.cpu())
    with pytest.raises(RuntimeError, match="derivative"):
        call(k=k.clone().requires_grad_(True))
    assert hb.append_to_cache(k[:0], k[:0], cu[:1], c["k"], c["v"], c["table"][:0], c["cache_lens"][:0]).shape == (0,)


# ------------------------------------------------------------------------------------------------------------------ select
def selected(weights, lens, budget, sink, recent):
    """Definition, on the host: sorted by weight (NaN first), then by position."""
    w = weights.cpu().tolist()
    kept = torch.full((len(w), len(w[0]), budget), -1, dtype=torch.int32)
    for b, heads in enumerate(w):
        n = max(0, min(lens[b], len(heads[0])))
        for h, row in enumerate(heads):
            if n <= budget:
                stays = range(n)
            else:
                middle = sorted(range(sink, n - recent), key=lambda i: (-math.inf if math.isnan(row[i]) else -row[i], 0 if math.isnan(row[i]) else 1, i))
                stays = sorted([*range(sink), *middle[:budget - sink - recent], *range(n - recent, n)])
            kept[b, h, :len(stays)] = torch.tensor(list(stays), dtype=torch.int32)
    return kept


def _check_select(w, lens, budget, sink, recent):
    import hbsattn_b200 as hb
    kept, kept_lens = hb.select_keys(w, torch.tensor(lens, dtype=torch.int32, device="cuda"), budget, sink, recent)
    cut = [max(0, min(n, w.shape[2])) for n in lens]
    assert kept_lens.tolist() == [min(n, budget) for n in cut] and kept_lens.dtype == kept.dtype == torch.int32
    assert torch.equal(kept.cpu(), selected(w, lens, budget, sink, recent))


LENS = [0, 1, 31, 32, 33, 500, 1024, 1025, 3000]


@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (32, 4, 8), (64, 32, 32), (100, 0, 7), (1000, 16, 64), (5000, 3, 5)])
@pytest.mark.parametrize("kind", ["spread", "tied", "equal", "special", "tiny"])
def test_select(kind, budget, sink, recent):
    g = torch.Generator().manual_seed(6)
    w = torch.exp(3 * torch.randn(len(LENS), 2, 3000, generator=g))
    if kind == "tied":
        w = torch.randint(0, 4, w.shape, generator=g).float()
    elif kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "special":                           # signs, both zeros, infinities, NaN of both signs
        values = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, -math.nan, 1e-42, -1e-42])
        w = values[torch.randint(0, len(values), w.shape, generator=g)]
    elif kind == "tiny":                              # neighbouring numbers, which differ in the last bits alone
        w = (torch.randint(0, 600, w.shape, generator=g).to(torch.int32) + 0x3F800000).view(torch.float32)
    _check_select(w.cuda(), LENS, budget, sink, recent)


@pytest.mark.parametrize("n,budget", [(70001, 4096), (300000, 70000)])
def test_select_long(n, budget):
    g = torch.Generator().manual_seed(7)
    w = torch.exp(2 * torch.randn(2, 1, n, generator=g)) * (torch.rand(2, 1, n, generator=g) < 0.5)
    _check_select(w.cuda(), [n, n - 1234], budget, 4, 1000)


def test_select_strides_lengths_and_graph():
    import hbsattn_b200 as hb
    g = torch.Generator().manual_seed(8)
    w = torch.randn(3, 4, 257, generator=g).cuda()
    _check_select(w[..., 1:200], [300, -5, 199], 50, 2, 3)
    _check_select(w.transpose(0, 1)[:, :, 5:], [100, 252, 1000, 51], 50, 2, 3)
    _check_select(w.permute(2, 1, 0).contiguous().permute(2, 1, 0), [100, 252, 51], 50, 2, 3)
    lens = torch.tensor([257, 200, 60], device="cuda")
    hb.select_keys(w, lens, 50)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, _ = hb.select_keys(w, lens.int(), 50)
    for seed in range(3):
        w.copy_(torch.randn(3, 4, 257, generator=g))
        graph.replay()
        assert torch.equal(kept.cpu(), selected(w, [257, 200, 60], 50, 0, 0))


def test_select_refusals():
    import hbsattn_b200 as hb
    w, lens = torch.rand(2, 2, 64, device="cuda"), torch.tensor([3, 64], device="cuda")
    for args in ((w.half(), lens, 4), (w[0], lens, 4), (w, lens[:1], 4), (w, lens, 0), (w, lens, 4, 3, 2), (w, lens, 4, -1, 2), (w, lens, 4, 1, -2), (w[..., :0], lens, 4),
                 (w, lens.float(), 4)):
        with pytest.raises(AssertionError):
            hb.select_keys(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        hb.select_keys(w, lens.cpu(), 4)
    with pytest.raises(RuntimeError, match="derivative"):
        hb.select_keys(w.clone().requires_grad_(True), lens, 4)


# ------------------------------------------------------------------------------------------------------------------ compact
@pytest.mark.parametrize("budget", [1, 40, 100, 700])
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_compact(kind, budget):
    import hbsattn_b200 as hb
    dtype, hk, d, page, layout = kind
    lens = [0, 1, 64, 65, 300, 1500]
    c = make_cache(9, lens, hk, d, page, dtype, layout=layout)
    capacity = c["table"].shape[1] * page
    w = torch.exp(torch.randn(len(lens), hk, capacity + 3, generator=torch.Generator().manual_seed(10))).cuda()
    sink, recent = min(4, budget // 2), min(16, budget // 3)
    kept, kept_lens = hb.select_keys(w[..., :capacity], c["cache_lens"], budget, sink, recent)
    want, want_w = [c["k"].clone(), c["v"].clone()], w.clone()
    for b, n in enumerate(lens):
        m = min(n, budget)
        want_w[b, :, :n] = 0
        for h in range(hk):
            src = kept[b, h, :m].long()
            to, of = _at(c, b, torch.arange(m)), _at(c, b, src)
            for new, old in zip(want, (c["k"], c["v"])):
                new[to[0], to[1], h] = old[of[0], of[1], h]
            want_w[b, h, :m] = w[b, h, src]
    assert hb.compact_cache(c["k"], c["v"], c["table"], c["cache_lens"], kept, kept_lens, key_weights=w) is None
    assert same(c["k"], want[0]) and same(c["v"], want[1]) and same(w, want_w)


def test_compact_long_rows_again_and_again():
    """In place: rows move down over rows that have been read already, and over nothing else, in every one of many orders."""
    import hbsattn_b200 as hb
    lens = [30000, 20011]
    c = make_cache(11, lens, 2, 64, 16, torch.bfloat16, fill=0.0)
    g = torch.Generator(device="cuda").manual_seed(12)
    for budget in (17000, 9001, 2500):
        w = torch.rand(2, 2, c["table"].shape[1] * 16, generator=g, device="cuda")
        now = c["cache_lens"]
        kept, kept_lens = hb.select_keys(w, now, budget, 4, 100)
        rows = []
        for b in range(2):
            for h in range(2):
                at = _at(c, b, kept[b, h, :int(kept_lens[b])].long())
                rows.append([t[at[0], at[1], h].clone() for t in (c["k"], c["v"])])
        hb.compact_cache(c["k"], c["v"], c["table"], now, kept, kept_lens)
        for i, (rk, rv) in enumerate(rows):
            at = _at(c, i // 2, torch.arange(rk.shape[0]))
            assert same(c["k"][at[0], at[1], i % 2], rk) and same(c["v"][at[0], at[1], i % 2], rv)
        c["cache_lens"] = kept_lens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compact_out_of_range(dtype):
    """Entries that are no position of the sequence, and pages that do not exist, move nothing and touch nothing else."""
    import hbsattn_b200 as hb
    c = make_cache(13, [64, 64], 1, 64, 16, dtype, extra_pages=0)
    other = [t[c["table"][1].long()].clone() for t in (c["k"], c["v"])]
    table = c["table"].clone()
    table[0, 2] = c["k"].shape[0] + 5
    kept = torch.tensor([[[1, 20, 40, 50, 64, 2 ** 31 - 1, -2 ** 31, -1]], [[0, 1, 2, 3, -1, -1, -1, -1]]], dtype=torch.int32, device="cuda")
    want = [c["k"].clone(), c["v"].clone()]
    for j, src in ((0, 1), (1, 20), (3, 50)):
        to, of = _at(c, 0, [j]), _at(c, 0, [src])
        for new, old in zip(want, (c["k"], c["v"])):
            new[to] = old[of]
    hb.compact_cache(c["k"], c["v"], table, c["cache_lens"], kept, torch.tensor([100, 4], device="cuda"))
    assert same(c["k"], want[0]) and same(c["v"], want[1])
    for t, o in zip((c["k"], c["v"]), other):
        assert same(t[c["table"][1].long()], o)


def test_compact_refusals():
    import hbsattn_b200 as hb
    c = make_cache(14, [64, 64], 2, 64, 16, torch.bfloat16, extra_pages=0)
    kept = torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda")
    n, w = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 64, device="cuda")

    def call(k=c["k"], v=c["v"], kept=kept, n=n, w=w):
        return hb.compact_cache(k, v, c["table"], c["cache_lens"], kept, n, key_weights=w)
    call()
    for more in (dict(kept=kept[0]), dict(kept=kept[:, :1]), dict(kept=kept.float()), dict(kept=kept[..., :0]), dict(n=n[:1]), dict(w=w[..., :-1]), dict(w=w.half()),
                 dict(v=c["v"][:-1]), dict(k=c["k"][:1].expand(8, -1, -1, -1), v=c["v"][:1].expand(8, -1, -1, -1)), dict(w=w[:, :1].expand(-1, 2, -1))):
        with pytest.raises(AssertionError):
            call(**more)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(kept=kept.cpu())
    with pytest.raises(RuntimeError, match="derivative"):
        call(w=w.clone().requires_grad_(True))


def test_what_autograd_has_saved_is_known_to_have_changed():
    """The in-place operators count as in-place operators, on the native path and on the general one (odd types of the lengths)."""
    import hbsattn_b200 as hb
    c = make_cache(15, [64, 64], 2, 64, 16, torch.bfloat16, extra_pages=1, room=1)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.rand(2, 2, c["table"].shape[1] * 16, device="cuda")
    kept, n = hb.select_keys(w, c["cache_lens"], 8)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    for lens in (c["cache_lens"], c["cache_lens"].long()):
        calls = [((c["k"], c["v"]), lambda: hb.append_to_cache(k, k, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), c["k"], c["v"], c["table"], lens)),
                 ((w,), lambda: hb.paged_attention(q, c["k"], c["v"], c["table"], lens, key_weights=w)),
                 ((c["k"], c["v"], w), lambda: hb.compact_cache(c["k"], c["v"], c["table"], lens, kept, n, key_weights=w))]
        for written, call in calls:
            x = torch.ones(written[0].shape, dtype=written[0].dtype, device="cuda", requires_grad=True)
            y = (x * written[0]).sum()
            before = [t._version for t in written]
            call()
            assert all(t._version > v for t, v in zip(written, before))
            with pytest.raises(RuntimeError, match="inplace"):
                y.backward()
    with torch.inference_mode():
        held = make_cache(16, [64], 2, 64, 16, torch.bfloat16, room=1)
        one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        assert hb.append_to_cache(k[:1], k[:1], one, held["k"], held["v"], held["table"], held["cache_lens"]).tolist() == [65]
