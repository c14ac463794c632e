"""Selection of keys where weights crowd: values that differ in their lowest bits only, in few bits, by many orders, and equal ones, around the sizes
at which the kernel changes its ways (256, 1024, 2048, 8192, 32768 positions), against a stable sort."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def weights_of(kind, n, g):
    i = torch.randperm(n, generator=g)
    if kind == "low bits":
        return (0x3f800000 + i).to(torch.int32).view(torch.float32)
    if kind == "few values":
        return (i % 7).float()
    if kind == "runs":                                 # many of a few neighbouring numbers, others far away
        return torch.where(i % 3 == 0, 1e-30 * i.float(), (0x40000000 + i % 5).to(torch.int32).view(torch.float32))
    if kind == "orders":
        return torch.exp(40 * torch.randn(n, generator=g))
    if kind == "signs":
        return torch.where(i % 4 == 0, torch.tensor(0.0), torch.where(i % 4 == 1, torch.tensor(-0.0), torch.randn(n, generator=g)))
    assert kind == "one bin"                           # the first digit tells nothing apart but one
    w = 1 + i.float() * 2.0 ** -23
    w[int(i[0])] = 3e38
    return w


@pytest.mark.parametrize("kind", ["low bits", "few values", "runs", "orders", "signs", "one bin"])
@pytest.mark.parametrize("n", [31, 255, 256, 257, 1023, 1025, 2049, 8192, 8193, 20000, 33000, 140000])
def test_crowded_weights(kind, n):
    import hbsattn_b200 as hb
    g = torch.Generator().manual_seed(n)
    rows = 3
    w = torch.stack([weights_of(kind, n, g) for _ in range(rows)])
    lens = torch.tensor([n, n - 1, max(n // 2, 1)], dtype=torch.int32)
    for budget, sink, recent in ((n // 8 + 2, 1, 1), (n // 2, 0, 3), (max(n - 3, 1), 0, 0), (5, 2, 3)):
        kept, kept_lens = hb.select_keys(w[:, None].cuda(), lens.cuda(), budget, sink, recent)
        for b in range(rows):
            m = int(lens[b])
            if m <= budget:
                want = torch.arange(m)
            else:
                x = w[b, sink:m - recent] + 0.0        # the order of numbers: both zeros alike
                heavy = torch.sort(x, descending=True, stable=True).indices[:budget - sink - recent] + sink
                want = torch.cat([torch.arange(sink), heavy.sort().values, torch.arange(m - recent, m)])
            assert int(kept_lens[b]) == want.numel()
            assert torch.equal(kept[b, 0, :want.numel()].cpu().long(), want)
            assert bool((kept[b, 0, want.numel():] == -1).all())


def test_not_a_number_stays_first():
    import hbsattn_b200 as hb
    for n in (500, 3000, 20000):
        w = torch.rand(1, 1, n, generator=torch.Generator().manual_seed(n))
        w[0, 0, 7::50] = math.nan
        w[0, 0, 9::50] = math.inf
        count = (n - 7 + 49) // 50
        kept, _ = hb.select_keys(w.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), count, 0, 0)
        assert torch.equal(kept[0, 0].cpu().long(), torch.arange(7, n, 50))
