"""Calls at the ends of what the paged cache's operators allow: very large groups, nothing to do, lists that do not ascend, the same position
twice, rows beyond the budget, two graphs on two streams."""
import math

import pytest
import torch

from cache_helpers import make_cache
from test_gpu_paged_attention import _check, _q, _weights_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [33, 257, 1100])
def test_very_large_groups(group, dtype):
    import hbsattn_b200 as hb
    lens, d, page = [70, 0, 260], 64, 16
    c = make_cache(41, lens, 1, d, page, dtype)
    q = _q(42, 3, group, d, dtype)
    start = torch.zeros(3, 1, c["table"].shape[1] * page).cuda()
    w = start.clone()
    out, lse = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w, return_lse=True)
    weights, size = _check(q, c, out, lse)
    # sums over the heads: one rounding of fp32 more for every head
    _weights_check(w, start, weights, d, max(lens) + group, size)


@pytest.mark.parametrize("family", ["auto", "generic"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_key_weights_of_nothing(dtype, family):
    import hbsattn_b200 as hb
    k = torch.randn(50, 2, 64).to(dtype).cuda()
    cu = torch.tensor([0, 50], dtype=torch.int32).cuda()
    hb.set_kernel_family(family)
    try:
        none = torch.tensor([0, 0], dtype=torch.int32).cuda()
        w = hb.attention_key_weights(k[:0], k, torch.empty(0, 2).cuda(), none, cu, torch.ones(2, 1, 1, dtype=torch.bool).cuda(), 16, 64, False)
        assert w.shape == (50, 2) and not w.any()
        # rows that see no key at all
        lse = torch.full((50, 2), -math.inf).cuda()
        w = hb.attention_key_weights(k, k, lse, cu, cu, torch.ones(2, 1, 1, dtype=torch.bool).cuda(), 64, 64, True)
        assert not w.any()
        w = hb.attention_key_weights(k, k, lse + 1, cu, cu, torch.zeros(2, 1, 1, dtype=torch.bool).cuda(), 64, 64, True)
        assert not w.any()
    finally:
        hb.set_kernel_family("auto")


def test_append_with_lists_that_do_not_ascend():
    """What they say is nonsense, but nothing outside the sequences' pages is written."""
    import hbsattn_b200 as hb
    c = make_cache(43, [5, 9, 0], 2, 64, 16, torch.bfloat16, fill=0.0)
    used = torch.zeros(c["k"].shape[0], dtype=torch.bool, device="cuda")
    used[c["table"].long().clamp(0, c["k"].shape[0] - 1).flatten()] = True
    k = torch.ones(20, 2, 64, dtype=torch.bfloat16, device="cuda")
    for cu in ([0, 12, 4, 20], [20, 10, 5, 0], [-5, 3, 30, 90], [0, -1, -2, 7]):
        before = [c["k"].clone(), c["v"].clone()]
        hb.append_to_cache(k, k, torch.tensor(cu, dtype=torch.int32).cuda(), c["k"], c["v"], c["table"], c["cache_lens"])
        torch.cuda.synchronize()
        assert torch.equal(c["k"][~used], before[0][~used]) and torch.equal(c["v"][~used], before[1][~used])


def test_compact_with_the_same_position_twice():
    import hbsattn_b200 as hb
    c = make_cache(44, [100, 40], 2, 64, 16, torch.bfloat16)
    kept = torch.tensor([[3, 3, 7, 7, 7, 90], [1, 2, 2, 39, 39, 200]], dtype=torch.int32).cuda()[:, None].repeat(1, 2, 1).contiguous()
    lens = torch.tensor([6, 5], dtype=torch.int32).cuda()
    at = lambda b, i: (c["table"][b].long()[i // 16], i % 16)
    want = [[t[at(b, kept[b, 0, :int(lens[b])].long())].clone() for b in range(2)] for t in (c["k"], c["v"])]
    hb.compact_cache(c["k"], c["v"], c["table"], c["cache_lens"], kept, lens)
    for t, rows in zip((c["k"], c["v"]), want):
        for b in range(2):
            assert torch.equal(t[at(b, torch.arange(int(lens[b]), device="cuda"))], rows[b])


def test_two_graphs_on_two_streams():
    """Each graph has workspaces of its own: replayed side by side they give what they give alone."""
    import hbsattn_b200 as hb
    made = []
    for seed, lens, d, dtype in ((45, [9000, 40, 0], 128, torch.bfloat16), (46, [300, 7000], 64, torch.float32)):
        c = make_cache(seed, lens, 2, d, 16, dtype)
        q = _q(seed + 10, len(lens), 4, d, dtype)
        w = torch.zeros(len(lens), 2, c["table"].shape[1] * 16).cuda()

        def step(c=c, q=q, w=w):
            w.zero_()
            out = hb.paged_attention(q, c["k"], c["v"], c["table"], c["cache_lens"], key_weights=w)
            kept, kept_lens = hb.select_keys(w, c["cache_lens"], 128, 4, 16)
            return out, w, kept, kept_lens

        want = [x.clone() for x in step()]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            with torch.cuda.graph(graph, stream=stream):
                got = step()
        made.append((stream, graph, got, want, step))      # step keeps the graph's inputs
    for _ in range(30):
        for stream, graph, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in made:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
