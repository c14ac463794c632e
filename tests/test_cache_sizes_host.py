"""Sizes beyond 31 bits are refused on the host, before any launch."""
import ctypes

import pytest
import torch

FAKE = 0x1000
BIG = 2 ** 31


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


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _int(*shape, dtype=torch.int32):
    return _meta(*shape, dtype=dtype)


@pytest.fixture
def anywhere(monkeypatch):
    """The checks of shapes and types alone: they come before anything that needs the device."""
    from hbsattn_b200 import paged_cache
    monkeypatch.setattr(paged_cache, "_same_device", lambda *tensors: None)
    return paged_cache


CALLS = {
    "num_pages": lambda m: m.paged_attention(_meta(2, 4, 8), _meta(BIG, 16, 2, 8), _meta(BIG, 16, 2, 8), _int(2, 4), _int(2)),
    "nhead_k": lambda m: m.paged_attention(_meta(2, BIG, 8), _meta(1, 16, BIG, 8), _meta(1, 16, BIG, 8), _int(2, 4), _int(2)),
    "batch": lambda m: m.paged_attention(_meta(BIG, 4, 8), _meta(9, 16, 2, 8), _meta(9, 16, 2, 8), _int(BIG, 4), _int(BIG)),
    "nhead_q": lambda m: m.paged_attention(_meta(2, BIG, 8), _meta(9, 16, 2, 8), _meta(9, 16, 2, 8), _int(2, 4), _int(2)),
    "k_block_size": lambda m: m.paged_attention(_meta(2, 4, 8), _meta(9, 16, 2, 8), _meta(9, 16, 2, 8), _int(2, 4), _int(2), block_mask=_int(2, 2, 4, dtype=torch.bool),
                                                k_block_size=2 * BIG + 16),
    "num_k_block": lambda m: m.paged_attention(_meta(2, 4, 8), _meta(9, 16, 2, 8), _meta(9, 16, 2, 8), _int(2, 4), _int(2), block_mask=_int(2, 2, 2 * BIG + 4, dtype=torch.bool),
                                               k_block_size=16),
    "total": lambda m: m.append_to_cache(_meta(2 * BIG + 1, 2, 8), _meta(2 * BIG + 1, 2, 8), _int(3), _meta(9, 16, 2, 8), _meta(9, 16, 2, 8), _int(2, 4), _int(2)),
    "budget": lambda m: m.select_keys(_meta(2, 2, 64, dtype=torch.float32), _int(2), 2 * BIG + 5),
    "budget of kept": lambda m: m.compact_cache(_meta(9, 16, 2, 8), _meta(9, 16, 2, 8), _int(2, 4), _int(2), _int(2, 2, 2 * BIG + 5), _int(2)),
    "q_block_size": lambda m: m._key_weights(_meta(5, 4, 8), _meta(5, 2, 8), _meta(5, 4, dtype=torch.float32), _int(2), _int(2), _int(2, 1, 1, dtype=torch.bool), None, 1, 1,
                                             2 * BIG + 16, 64, True, None),
    "num_q_block": lambda m: m._key_weights(_meta(5, 4, 8), _meta(5, 2, 8), _meta(5, 4, dtype=torch.float32), _int(2), _int(2), None, None, 2 * BIG + 1, 1, 64, 64, True, None),
}


@pytest.mark.parametrize("what", CALLS)
def test_sizes_beyond_31_bits(anywhere, what):
    with pytest.raises(AssertionError, match=f"{what.split()[0]} must fit 31 bits"):
        CALLS[what](anywhere)


def test_complex_numbers_are_no_integers(anywhere):
    c, k = _int(2, dtype=torch.complex64), _meta(9, 16, 2, 8)
    for call in (lambda: anywhere.paged_attention(_meta(2, 4, 8), k, k, _int(2, 4), c), lambda: anywhere.select_keys(_meta(2, 2, 64, dtype=torch.float32), c, 4),
                 lambda: anywhere.compact_cache(k, k, _int(2, 4), _int(2), _int(2, 2, 3), c)):
        with pytest.raises(AssertionError, match="integer"):
            call()
