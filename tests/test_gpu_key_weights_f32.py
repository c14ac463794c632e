"""Key weights on the CUDA cores: row tiles strung together from q-blocks, rows split over clusters, more q-blocks than one look takes, and loads
by 16 bytes and by elements, against the definition in 64 bits."""
import pytest
import torch

from helpers import make_problem
from test_gpu_key_weights import check, exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [4, 64, 72, 128, 130, 256])
@pytest.mark.parametrize("hq,hk,qbs,kbs,causal", [(3, 3, 16, 16, True), (8, 2, 48, 80, False), (6, 1, 112, 64, True), (20, 4, 16, 272, True)])
def test_shapes(hq, hk, qbs, kbs, causal, d):
    import hbsattn_b200 as hb
    pr = make_problem(91, [403, 1, 250, 64], [403, 90, 250, 1], hq, hk, d, qbs, kbs, causal, torch.float32, 0.5, None)
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], qbs, kbs, causal)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], *rest)
    w = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
    assert hb.last_status()[0] == 0
    want, size = exact(pr, pr["q"], pr["k"], lse)
    check(pr, w, want, size, lse, d, hq // hk)
    assert torch.equal(w, hb.attention_key_weights(pr["q"], pr["k"], lse, *rest))
    wide = torch.zeros(pr["q"].shape[0], hq, 2 * d, device="cuda")[:, :, ::2]     # columns apart: no 16-byte units
    wide.copy_(pr["q"])
    assert torch.equal(w, hb.attention_key_weights(wide, pr["k"], lse, *rest))


@pytest.mark.parametrize("causal", [True, False])
def test_many_q_blocks(causal):
    """2100 q-blocks of 16 rows past the keys of a short and of a long sample."""
    import hbsattn_b200 as hb
    pr = make_problem(92, [33600, 700], [150, 700], 1, 1, 64, 16, 64, causal, torch.float32, 0.7, None)
    rest = (pr["cu_q"], pr["cu_k"], pr["mask"], 16, 64, causal)
    _, lse = hb.HBSAttention_with_lse(pr["q"], pr["k"], pr["v"], *rest)
    w = hb.attention_key_weights(pr["q"], pr["k"], lse, *rest)
    want, size = exact(pr, pr["q"], pr["k"], lse)
    check(pr, w, want, size, lse, 64, 1)
