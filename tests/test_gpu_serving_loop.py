"""The operators together, as a serving loop with eviction uses them: prompts through block-sparse attention, their keys into the cache
and their weights kept, decoding steps that add to the weights, an eviction in the middle, more steps - against the same
loop on plain packed tensors in 64 bits.  Which keys stay is decided by 32-bit weights, so the plain loop takes the positions that the
operator has chosen, after checking that its choice is right for the plain weights up to their error."""
import pytest
import torch

from cache_helpers import attention_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hq,hk,d,page", [(torch.bfloat16, 8, 2, 128, 16), (torch.float16, 12, 4, 64, 64), (torch.float32, 4, 4, 32, 8)])
def test_prefill_decode_evict(dtype, hq, hk, d, page):
    import hbsattn_b200 as hb
    lens, steps, budget, sink, recent = [300, 77, 150, 1], 20, 96, 4, 24
    batch, group, block, dev = len(lens), hq // hk, 64, "cuda"
    cu_list = [0]
    for n in lens:
        cu_list.append(cu_list[-1] + n)
    g = torch.Generator().manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dtype).cuda()
    q, k, v = normal(cu_list[-1], hq, d), normal(cu_list[-1], hk, d), normal(cu_list[-1], hk, d)
    cu = torch.tensor(cu_list, dtype=torch.int32, device=dev)
    n_block = sum(-(-n // block) for n in lens)
    mask = (torch.rand(hk, n_block, n_block, generator=g) < 0.5).to(dev)
    mask |= torch.eye(n_block, dtype=torch.bool, device=dev)
    rest = (cu, cu, mask, block, block, True)
    out, lse = hb.HBSAttention_with_lse(q, k, v, *rest)
    prompt_weights = hb.attention_key_weights(q, k, lse, *rest)

    capacity = -(-(max(lens) + steps) // page) * page
    table = torch.randperm(batch * capacity // page + 3, generator=g)[:batch * capacity // page].to(torch.int32).reshape(batch, -1).cuda()
    kc, vc = (torch.zeros(batch * capacity // page + 3, page, hk, d, dtype=dtype, device=dev) for _ in "kv")
    cache_lens = hb.append_to_cache(k, v, cu, kc, vc, table, torch.zeros(batch, dtype=torch.int32, device=dev))
    assert cache_lens.tolist() == lens
    w = torch.zeros(batch, hk, capacity, device=dev)
    for b, n in enumerate(lens):
        w[b, :, :n] = prompt_weights[cu_list[b]:cu_list[b + 1]].t()

    # the plain loop: per sequence and kv-head a list of keys, values and weights
    plain = [[[k[cu_list[b]:cu_list[b + 1], h].double(), v[cu_list[b]:cu_list[b + 1], h].double(), w[b, h, :lens[b]].double()] for h in range(hk)]
             for b in range(batch)]
    one = torch.arange(batch + 1, dtype=torch.int32, device=dev)

    def step():
        nonlocal cache_lens
        q1, k1, v1 = normal(batch, hq, d), normal(batch, hk, d), normal(batch, hk, d)
        cache_lens = hb.append_to_cache(k1, v1, one, kc, vc, table, cache_lens)
        got = hb.paged_attention(q1, kc, vc, table, cache_lens, key_weights=w)
        for b in range(batch):
            for h in range(hk):
                pk, pv, pw = plain[b][h]
                pk, pv, pw = torch.cat([pk, k1[b, h:h + 1].double()]), torch.cat([pv, v1[b, h:h + 1].double()]), torch.cat([pw, pw.new_zeros(1)])
                rows = q1[b, h * group:(h + 1) * group].double()
                p = torch.softmax(rows @ pk.T * d ** -0.5, dim=-1)
                size = float((rows.abs() @ pk.abs().T).max()) * d ** -0.5
                want = p @ pv
                tol = attention_tolerance(dtype, d, pk.shape[0], want, p @ pv.abs(), size)
                assert bool(((got[b, h * group:(h + 1) * group].double() - want).abs() <= tol).all())
                plain[b][h] = [pk, pv, pw + p.sum(dim=0)]
    for _ in range(steps // 2):
        step()
    kept, kept_lens = hb.select_keys(w, cache_lens, budget, sink, recent)
    hb.compact_cache(kc, vc, table, cache_lens, kept, kept_lens, key_weights=w)
    for b in range(batch):
        n, m = int(cache_lens[b]), int(kept_lens[b])
        assert m == min(n, budget)
        for h in range(hk):
            stay = kept[b, h, :m].long()
            pk, pv, pw = plain[b][h]
            gone = torch.ones(n, dtype=torch.bool, device=dev).index_fill(0, stay, False)
            if bool(gone.any()):                       # no key that went has more weight than one that stayed for its weight
                chosen = stay[(stay >= sink) & (stay < n - recent)]
                assert float(pw[gone].max()) <= float(pw[chosen].min()) * (1 + 1e-4)
                assert set(range(sink)) | set(range(n - recent, n)) <= set(stay.tolist())
            plain[b][h] = [pk[stay], pv[stay], pw[stay]]
            assert bool(((w[b, h, :m].double() - pw[stay]).abs() <= 1e-4 * pw[stay]).all()) and not w[b, h, m:].any()
    cache_lens = kept_lens
    for _ in range(steps // 2):
        step()
