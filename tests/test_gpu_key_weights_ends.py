"""Key weights at the ends of what the arguments allow, and beyond: blocks larger than everything that is packed, samples that reach beyond the tensors."""
import pytest
import torch

from helpers import make_problem
from test_gpu_key_weights import check, exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("family", ["auto", "generic"])
@pytest.mark.parametrize("qbs,kbs", [(2 ** 30, 2 ** 30), (2 ** 28, 64), (48, 2 ** 27 + 16), (2 ** 31 - 16, 2 ** 31 - 16)])
@pytest.mark.parametrize("hq,hk,d,causal,dtype", [(16, 2, 64, True, torch.bfloat16), (3, 3, 128, False, torch.float16), (4, 1, 32, True, torch.float32)])
def test_blocks_larger_than_the_packed_rows(hq, hk, d, causal, dtype, qbs, kbs, family):
    """One block a sample, as with any block size that holds the samples; the workspace goes by the rows."""
    import hbsattn_b200 as hb
    lens_q, lens_k = [70, 3, 150], [70, 128, 33]
    within = (min(qbs, 256), min(kbs, 256))               # (no sample has more than 256 rows)
    pr = make_problem(1, lens_q, lens_k, hq, hk, d, *within, causal, dtype, 0.8, None)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], pr["cu_q"], pr["cu_k"], pr["mask"], *within, causal)
    hb.set_kernel_family(family)
    try:
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        w = hb.attention_key_weights(pr["q"], pr["k"], lse, pr["cu_q"], pr["cu_k"], pr["mask"], qbs, kbs, causal)
        assert hb.last_status()[0] == 0
        assert torch.cuda.max_memory_allocated() - before < 8 << 20
    finally:
        hb.set_kernel_family("auto")
    want, size = exact(pr, pr["q"], pr["k"], lse)
    check(pr, w, want, size, lse, d, hq // hk)


def test_the_size_of_the_workspace_goes_by_the_rows():
    import ctypes

    from hbsattn_b200 import _lib
    lib = _lib.load()
    a = _lib.KeyWeightsArgs()
    a.struct_bytes = ctypes.sizeof(a)
    f = a.fwd
    f.num_q_block, f.num_k_block, f.nhead_q, f.total_q, f.total_k, f.k_block_size = 3, 3, 16, 223, 231, 64
    sizes = []
    for f.q_block_size in (256, 1024, 2 ** 30, 2 ** 31 - 16):
        sizes.append(lib.hbsa_key_weights_workspace_bytes(ctypes.byref(a)))
    assert len(set(sizes)) == 1 and sizes[0] < 1 << 20
    f.q_block_size, f.total_q = 1024, 0                   # not known yet: enough for any
    assert lib.hbsa_key_weights_workspace_bytes(ctypes.byref(a)) >= 3 * 1024 * 16 * 4


@pytest.mark.parametrize("family", ["auto", "generic"])
@pytest.mark.parametrize("kbs", [64, 128])
@pytest.mark.parametrize("hq,hk,d,causal,dtype", [(8, 2, 64, True, torch.bfloat16), (3, 3, 128, False, torch.float16), (4, 1, 32, True, torch.float32)])
def test_samples_that_reach_beyond_the_tensors(hq, hk, d, causal, dtype, kbs, family):
    """Rows and keys before the first and behind the last one that is there: not read, not written, and without weight."""
    import hbsattn_b200 as hb
    front, behind, qbs = 37, 45, 64
    lens = [150, 70, 200]
    pr = make_problem(3, lens, lens, hq, hk, d, qbs, kbs, causal, dtype, 0.6, None)
    total = sum(lens)
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], qbs, kbs, causal)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], *rest)
    lse[:front] = lse[total - behind:] = float("-inf")        # the whole problem without the rows that will be missing
    hb.set_kernel_family(family)
    try:
        want = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
        cut = slice(front, total - behind)
        cu = pr["cu_q"] - front
        got = hb.attention_key_weights(pr["q"][cut].clone(), pr["k"][cut].clone(), lse[cut].clone(), cu, cu, *rest[2:])
        assert hb.last_status()[0] == 0
        assert torch.equal(got, want[cut])
        none = torch.zeros_like(pr["mask"])                   # nothing active: zeros for the keys that are there
        assert not hb.attention_key_weights(pr["q"][cut].clone(), pr["k"][cut].clone(), lse[cut].clone(), cu, cu, none, *rest[3:]).any()
    finally:
        hb.set_kernel_family("auto")
