"""The paged cache's entry points on a machine without a GPU: struct mirrors, workspace sizes, and refusals before any launch."""
import ctypes

import pytest

FAKE = 0x1000


@pytest.fixture(scope="module")
def lib():
    from hbsattn_b200 import _lib
    return _lib.load()


def _cache(_lib, **over):
    c = _lib.Cache()
    c.k = c.v = c.block_table = c.lens = FAKE
    c.num_pages, c.page_size, c.max_pages, c.batch, c.nhead_k, c.headdim, c.dtype = 10, 16, 4, 3, 2, 64, _lib.HBSA_DTYPE_BF16
    c.table_stride = 4
    for i, s in enumerate((16 * 2 * 64, 2 * 64, 64, 1)):
        c.k_stride[i] = c.v_stride[i] = s
    for name, value in over.items():
        setattr(c, name, value)
    return c


def _args(kind, cache=None, **over):
    from hbsattn_b200 import _lib
    a = getattr(_lib, kind)()
    a.struct_bytes = ctypes.sizeof(a)
    fields = {name for name, *_ in a._fields_}
    if "cache" in fields:
        a.cache = _cache(_lib, **(cache or {}))
    values = dict(q=FAKE, o=FAKE, k=FAKE, v=FAKE, cu_seqlens=FAKE, new_lens=FAKE, status=FAKE, total=5, workspace=FAKE, workspace_bytes=1 << 40, nhead_q=4,
                  use_default_scale=1, key_weights=FAKE, lens=FAKE, kept=FAKE, kept_lens=FAKE, batch=3, nhead_k=2, max_len=64, budget=8, n_sink=1, n_recent=1)
    if kind == "PagedAttentionArgs":
        values["key_weights"] = None
        for i, s in enumerate((4 * 64, 64, 1)):
            a.q_stride[i] = a.o_stride[i] = s
    for name, value in {**values, **over}.items():
        if name in fields:
            setattr(a, name, value)
        else:
            assert name not in over, name
    return a


NAMES = {"AppendArgs": "hbsa_append_to_cache", "PagedAttentionArgs": "hbsa_paged_attention", "SelectKeysArgs": "hbsa_select_keys", "CompactArgs": "hbsa_compact_cache"}

BAD_CACHES = [(dict(k=None), -1), (dict(lens=None), -1), (dict(block_table=None), -1), (dict(batch=0), -2), (dict(page_size=0), -2), (dict(num_pages=-1), -2),
              (dict(headdim=257), -2), (dict(max_pages=2 ** 30), -2), (dict(batch=2 ** 30), -2), (dict(dtype=7), -4)]


@pytest.mark.parametrize("kind", ["AppendArgs", "PagedAttentionArgs", "CompactArgs"])
@pytest.mark.parametrize("cache,code", BAD_CACHES)
def test_bad_caches_are_refused(lib, kind, cache, code):
    from hbsattn_b200 import _lib
    assert getattr(lib, NAMES[kind])(ctypes.byref(_args(kind, cache)), None) == code
    assert _lib.last_error()


@pytest.mark.parametrize("kind,over,code", [
    ("AppendArgs", dict(struct_bytes=8), -8), ("AppendArgs", dict(cu_seqlens=None), -1), ("AppendArgs", dict(status=None), -1), ("AppendArgs", dict(total=-1), -2),
    ("AppendArgs", dict(k=None), -1),
    ("PagedAttentionArgs", dict(struct_bytes=8), -8), ("PagedAttentionArgs", dict(q=None), -1), ("PagedAttentionArgs", dict(nhead_q=3), -2),
    ("PagedAttentionArgs", dict(impl=9), -4), ("PagedAttentionArgs", dict(workspace_bytes=100), -5), ("PagedAttentionArgs", dict(workspace=FAKE + 8), -5),
    ("PagedAttentionArgs", dict(block_mask=FAKE, k_block_size=24, num_k_block=9), -3), ("PagedAttentionArgs", dict(block_mask=FAKE, k_block_size=16, num_k_block=3), -2),
    ("PagedAttentionArgs", dict(impl=2, use_default_scale=0, softmax_scale=-1.0), -6),
    ("SelectKeysArgs", dict(struct_bytes=8), -8), ("SelectKeysArgs", dict(kept=None), -1), ("SelectKeysArgs", dict(budget=0), -2), ("SelectKeysArgs", dict(n_sink=8), -2),
    ("SelectKeysArgs", dict(n_recent=-1), -2), ("SelectKeysArgs", dict(max_len=2 ** 31 - 1), -2), ("SelectKeysArgs", dict(batch=2 ** 30), -2),
    ("CompactArgs", dict(struct_bytes=8), -8), ("CompactArgs", dict(kept_lens=None), -1), ("CompactArgs", dict(budget=0), -2),
])
def test_bad_arguments_are_refused(lib, kind, over, code):
    from hbsattn_b200 import _lib
    assert getattr(lib, NAMES[kind])(ctypes.byref(_args(kind, **over)), None) == code
    assert _lib.last_error()


def test_workspace_bytes(lib):
    def size(cache=None, **over):
        return lib.hbsa_paged_attention_workspace_bytes(ctypes.byref(_args("PagedAttentionArgs", cache, workspace=None, **over)))
    plain = size()
    assert 0 < plain < 16 << 20 and plain % 256 == 0
    assert size(dict(max_pages=1 << 20)) == plain                       # independent of the length
    assert size(key_weights=FAKE) >= plain + 4 * 3 * 4 * 64              # a score per key and q-head
    assert size(block_mask=FAKE, k_block_size=16, num_k_block=4) > plain
    assert size(nhead_q=3) == 0


def test_key_weights_arguments(lib):
    from hbsattn_b200 import _lib
    from test_abi_host import _args as forward_args
    a = _lib.KeyWeightsArgs()
    a.struct_bytes = ctypes.sizeof(a)
    a.fwd = forward_args(v=None, o=None)
    assert lib.hbsa_key_weights_workspace_bytes(ctypes.byref(a)) >= 64 * 4 * 4
    a.weights = a.partial_workspace = FAKE
    a.partial_workspace_bytes = 1 << 30
    assert lib.hbsa_key_weights(ctypes.byref(a), None) == -1 and "lse" in _lib.last_error()
    a.fwd.lse = FAKE
    a.partial_workspace_bytes = 8
    assert lib.hbsa_key_weights(ctypes.byref(a), None) == -5
    a.fwd = forward_args(nhead_q=3)
    assert lib.hbsa_key_weights(ctypes.byref(a), None) == -2
    a.struct_bytes = 8
    assert lib.hbsa_key_weights(ctypes.byref(a), None) == -8


def test_operators_refuse_cpu_tensors():
    import torch

    import hbsattn_b200 as hb
    cache = torch.zeros(2, 16, 1, 16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x, cu, w = torch.zeros(1, 1, 16), torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, 1, 32)
    mask = torch.ones(1, 1, 1, dtype=torch.bool)
    for call in (lambda: hb.append_to_cache(x, x, cu, cache, cache, table, lens), lambda: hb.paged_attention(x, cache, cache, table, lens),
                 lambda: hb.attention_key_weights(x, x, x[..., 0], cu, cu, mask, 16, 16, True), lambda: hb.select_keys(w, lens, 4),
                 lambda: hb.compact_cache(cache, cache, table, lens, table[None], lens)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_workspace_does_not_depend_on_addresses_and_strides(d, dtype):
    """A size that was asked for without tensors is enough for whichever kernel the tensors lead to."""

    from hbsattn_b200 import _lib
    lib = _lib.load()
    a = _lib.PagedAttentionArgs()
    a.struct_bytes = ctypes.sizeof(a)
    a.cache.num_pages, a.cache.page_size, a.cache.nhead_k, a.cache.headdim = 10, 16, 2, d
    a.cache.batch, a.cache.max_pages, a.cache.dtype, a.nhead_q, a.use_default_scale = 3, 4, dtype, 8, 1
    asked = lib.hbsa_paged_attention_workspace_bytes(ctypes.byref(a))
    a.cache.k = a.cache.v = a.q = a.o = 1 << 20
    for strides in ((16 * 2 * d, 2 * d, d, 1), (16 * 2 * (d + 1), 2 * (d + 1), d + 1, 1)):
        for i in range(4):
            a.cache.k_stride[i] = a.cache.v_stride[i] = strides[i]
        for i in range(3):
            a.q_stride[i] = a.o_stride[i] = strides[i + 1]
        assert lib.hbsa_paged_attention_workspace_bytes(ctypes.byref(a)) == asked > 0
