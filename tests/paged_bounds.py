"""Bounds of the decoding kernels' errors that are tight enough to notice one lost tile of 64 keys among tens of thousands."""
import torch

from cache_helpers import score_error


def chain(lens, heads_k, sms=148):
    """Terms that follow one another in a sum: the keys of a CTA's part of a row (as if one after the other), its warps, and the parts of a
    row, of which a quarter (of at most four for every SM) follow one another and then four to sixteen sums.  The tiles of all rows are cut into equal
    runs, of which there is at least one for every second SM."""
    runs = sms // 2
    tiles = sum(-(-n // 64) for n in lens) * heads_k
    parts = min(4 * sms, -(-max(lens) // 64) + 1)
    return 64 * (-(-tiles // runs)) + 8 + parts // 4 + 16


def out_bound(dtype, d, out, spread, squares, size, depth):
    """`spread`: sum of p |v|, `squares`: sum of (p v)^2.  The result is rounded once, by half a step at most.  Every p of 16 bits is off by half
    a step at most, one independently of the other: of such sums sqrt(sum (half p v)^2 / 3) is the standard deviation at most, of which
    eight times is taken (fp16 has half a step of 2^-11 down to 2^-28 of the largest p).  32 bits: the score's error in p and in the sum, sums
    of `depth` terms (2^-24 each, in O and in the sum), exponentials and the division."""
    half = torch.finfo(dtype).eps / 2
    c32 = 2 * score_error(d, size) + 2 * depth * 2.0 ** -24 + 2.0 ** -20
    tol = half * out.abs() * (1 + 2 * half) + c32 * spread + 2.0 ** -25
    return tol if dtype == torch.float32 else tol + 8 * half / 3 ** 0.5 * squares.sqrt()


def lse_bound(d, lse, size, depth):
    return score_error(d, size) + depth * 2.0 ** -24 + 2.0 ** -20 + lse.abs() * 2.0 ** -22
