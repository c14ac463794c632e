"""Sizes beyond 31 bits are refused on the host, before any launch."""
import ctypes

FAKE = 0x1000


def test_key_weights_of_blocks_beyond_31_bits():
    from hbsattn_b200 import _lib
    from test_abi_host import _args as forward_args
    lib = _lib.load()
    a = _lib.KeyWeightsArgs()
    a.struct_bytes = ctypes.sizeof(a)
    a.weights = a.partial_workspace = FAKE
    a.partial_workspace_bytes = 1 << 62
    a.fwd = forward_args(v=None, o=None, nhead_q=2, nhead_k=2, q_block_size=2 ** 30, total_q=2 ** 31 - 1)
    a.fwd.lse = FAKE
    assert lib.hbsa_key_weights(ctypes.byref(a), None) == -2 and "2^31 rows" in _lib.last_error()
