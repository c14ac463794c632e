"""The bounds of paged_bounds.py notice any tile of 64 keys that is left out or counted twice: on the definition in 64 bits, for the sizes of
test_gpu_paged_tight.py."""
import pytest
import torch

from paged_bounds import chain, lse_bound, out_bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,d,n", [(8, 64, 20000), (8, 128, 20000), (4, 256, 9000)])
def test_a_lost_or_doubled_tile_is_noticed(dtype, heads, d, n):
    g = torch.Generator().manual_seed(1)
    q = (2 * torch.randn(heads, d, generator=g)).to(dtype).double()
    k, v = (torch.randn(n, d, generator=g).to(dtype).double() for _ in "kv")
    x = d ** -0.5 * q @ k.T
    size = float((d ** -0.5 * q.abs() @ k.abs().T).max())
    p = torch.softmax(x, dim=-1)
    out, lse = p @ v, torch.logsumexp(x, dim=-1)
    depth = chain([n], 1)
    tol = out_bound(dtype, d, out, p @ v.abs(), (p ** 2) @ (v ** 2), size, depth)
    lse_tol = lse_bound(d, lse, size, depth)
    by_out = by_lse = tiles = 0
    for t in range(0, n, 64):
        share, part = p[:, t:t + 64].sum(dim=1, keepdim=True), p[:, t:t + 64] @ v[t:t + 64]
        for sign in (-1, 1):
            changed = (out + sign * part) / (1 + sign * share)
            by_out += bool(((changed - out).abs() > 2 * tol).any())      # whatever the kernel's own error is
            by_lse += bool((torch.log1p(sign * share[:, 0]).abs() > 2 * lse_tol).any())
            tiles += 1
    assert by_lse == tiles
    assert by_out >= 0.9 * tiles, f"{by_out} of {tiles}"
