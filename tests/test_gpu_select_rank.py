"""Selection where the last place falls among n weights of one first digit: around the number up to which they are ranked directly, distinct
and tied ones, in rows of every build of the kernel."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tied", ["distinct", "tied", "pairs"])
@pytest.mark.parametrize("length", [1500, 8000, 30000, 40000])
@pytest.mark.parametrize("n", [2, 127, 128, 129, 130, 257, 450])
def test_last_place_among_n(n, length, tied):
    import hbsattn_b200 as hb
    g = torch.Generator().manual_seed(n + length)
    low, high = 0x3A000000, 0x3FFFFFFF
    width = (high - low) // 2048                          # numbers of a first digit
    at = 1024 * width
    rows, budgets = [], []
    above = length // 3
    for r in range(3):
        among = {"distinct": torch.randperm(width // 2, generator=g)[:n], "tied": torch.zeros(n, dtype=torch.int64), "pairs": torch.arange(n) // 2}[tied]
        x = torch.cat([torch.randint(at + 2 * width, high - low, (above - 1,), generator=g), torch.tensor([high - low]), at + width // 4 + among,
                       torch.randint(1, at - width, (length - above - n - 1,), generator=g), torch.tensor([0])])
        rows.append((x + low)[torch.randperm(length, generator=g)].to(torch.int32).view(torch.float32))
    w = torch.stack(rows)
    lens = torch.full((3,), length, dtype=torch.int32).cuda()
    for place in (1, n // 2, n - 1, n):
        budget = above + place
        kept, kept_lens = hb.select_keys(w[:, None].cuda(), lens, budget)
        want = torch.sort(w, dim=1, descending=True, stable=True).indices[:, :budget].sort(dim=1).values
        assert kept_lens.tolist() == [budget] * 3
        assert torch.equal(kept[:, 0].cpu().long(), want), place
