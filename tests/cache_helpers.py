"""Paged caches for the tests, and what the cache operators compute, in 64 bits and one sequence at a time."""
import math

import torch

GARBAGE = float("nan")


def make_cache(seed, lens, nhead_k, headdim, page, dtype, spare=2, extra_pages=1, layout="nhd", fill=GARBAGE, room=0):
    """A cache whose sequences own shuffled pages.  What belongs to no position holds `fill`, what block_table holds behind a
    sequence's pages points nowhere.  `room`: positions for which pages are there beyond the lengths."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-(n + room) // page) for n in lens]
    width = max(max(pages), 1) + extra_pages
    order = torch.randperm(sum(pages) + spare, generator=g).to(torch.int32)
    table = torch.where(torch.rand(len(lens), width, generator=g) < 0.5, 2 ** 30, -7).to(torch.int32)
    shape = (order.numel(), page, nhead_k, headdim)
    k, v = (torch.full(shape, fill, dtype=dtype) for _ in "kv")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    c = dict(lens=list(lens), page=page, table_cpu=table)
    for b, n in enumerate(lens):
        pos = torch.arange(n)
        rows = table[b].long()[pos // page], pos % page
        for t in (k, v):
            t[rows] = torch.randn(n, nhead_k, headdim, generator=g).to(dtype)
    if layout == "hnd":                                  # heads outside the slots in memory
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    c.update(k=_cuda_as(k), v=_cuda_as(v), table=table.cuda(), cache_lens=torch.tensor(lens, dtype=torch.int32).cuda())
    return c


def _cuda_as(t):
    order = sorted(range(t.ndim), key=lambda i: -t.stride(i))
    back = [order.index(i) for i in range(t.ndim)]
    return t.permute(order).contiguous().cuda().permute(back)


def rows_of(c, cache, b, positions):
    """The rows of the given positions of sequence b."""
    positions = torch.as_tensor(positions, device=cache.device)
    table = c["table"][b].long()
    return cache[table[positions // c["page"]], positions % c["page"]]


def attention_exact(q, c, scale=None, mask=None, k_block=None, lens=None):
    """Per (sequence, q-head): output, log-sum-exp, sum of p |v| (what rounding P costs at most), weights of the keys summed over the
    group [batch, nhead_k, positions], and the largest sum of |q_i k_i| of a score, all in 64 bits."""
    batch, nhead_q, d = q.shape
    nhead_k = c["k"].shape[2]
    group, scale = nhead_q // nhead_k, d ** -0.5 if scale is None else scale
    lens = c["lens"] if lens is None else lens
    out, spread = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    weights = torch.zeros(batch, nhead_k, c["table"].shape[1] * c["page"], dtype=torch.float64, device=q.device)
    size = 0.0
    for b in range(batch):
        for h in range(nhead_k):
            pos = torch.arange(lens[b], device=q.device)
            if mask is not None:
                pos = pos[mask[b, h, pos // k_block]]
            if pos.numel() == 0:
                continue
            k, v = (rows_of(c, c[n], b, pos)[:, h].double() for n in "kv")
            heads = slice(h * group, (h + 1) * group)
            x = scale * q[b, heads].double() @ k.T
            size = max(size, float((abs(scale) * q[b, heads].double().abs() @ k.abs().T).max()))
            lse[b, heads] = torch.logsumexp(x, dim=-1)
            p = torch.softmax(x, dim=-1)
            out[b, heads], spread[b, heads] = p @ v, p @ v.abs()
            weights[b, h, pos] = p.sum(dim=0)
    return out, lse, spread, weights, size


def score_error(d, size):
    """How far a score of 32-bit products and sums can be off: d roundings (or cuts, 2^-23) of at most the sum of the products'
    magnitudes, and two of the score itself when it is scaled."""
    return (d + 2) * 2.0 ** -23 * size


def attention_tolerance(dtype, d, n, out, spread, size):
    """Bound of the output's error.  Roundings: the result (eps / 2 of it); P in 16 bits (eps / 2 of p |v|, for fp16 2^-25 at least per
    key); 32 bits: exp of a score that is off, once in p and once in the sum, the sum of n terms, and the exponential's own 2^-21."""
    half = torch.finfo(dtype).eps / 2
    c32 = 2 * score_error(d, size) + n * 2.0 ** -23 + 2.0 ** -20
    tol = half * out.abs() * (1 + 2 * half) + c32 * spread
    if dtype != torch.float32:
        tol = tol + half * spread
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -25 * 8 + 2.0 ** -24                # |v| < 8; results down to half a subnormal step
    return tol + 1e-30
