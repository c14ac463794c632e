"""Paged key-value cache: writing into it, attention of one new token per sequence over it, and eviction by attention weight.

The reference has no counterpart (its callers hand over packed keys and values, ``hbsattn/hbsa_interface.py:6-35``); these operators
continue where ``HBSAttention`` ends.  A serving loop with eviction::

    out, lse = HBSAttention_with_lse(q, k, v, cu, cu, mask, ...)                       # the prompts
    weights = attention_key_weights(q, k, lse, cu, cu, mask, ...)                      # [total, nhead_k]
    lens = append_to_cache(k, v, cu, k_cache, v_cache, block_table, lens)
    ...                                                                                # every new token:
    lens = append_to_cache(k1, v1, cu1, k_cache, v_cache, block_table, lens)
    out = paged_attention(q1, k_cache, v_cache, block_table, lens, key_weights=w)
    ...                                                                                # now and then:
    kept, kept_lens = select_keys(w, lens, budget, n_sink, n_recent)
    compact_cache(k_cache, v_cache, block_table, lens, kept, kept_lens, key_weights=w)
    lens = kept_lens

Layout: ``k_cache`` and ``v_cache`` are ``(num_pages, page_size, nhead_k, headdim)`` of any strides; position ``p`` of sequence ``b`` is
slot ``p % page_size`` of page ``block_table[b, p // page_size]`` (int32 ``[batch, max_pages]``), ``cache_lens`` (int32 ``[batch]``) says
how many positions are in use.  Entries of ``block_table`` behind a sequence's last page are not looked at.

The calls neither wait for the device nor read anything back: lengths outside the cache are cut, positions on pages that do not exist take
part in nothing, and ``last_status()`` then reports ``HBSA_STATUS_CACHE_BOUNDS`` (append and attention).  None of them has a
backward: tensors that require gradients are refused while gradients are recorded."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .hbsa_interface import _DTYPES, _IMPLS, _check_csr, _host, _prepare, _state, alloc_workspace, make_args


def _refuse_gradients(name, *tensors):
    for t in tensors:
        if t is not None and ((torch.is_grad_enabled() and t.requires_grad) or forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(f"{name} has no derivative: call it on detached tensors or under torch.no_grad()")


def _same_device(*tensors):
    if not all(t.is_cuda for t in tensors if t is not None):
        raise RuntimeError("hbsattn_b200 runs on CUDA tensors only (sm_100a); there is no CPU path")
    assert len({t.device for t in tensors if t is not None}) == 1, "all tensors must be on one device"


def _int32(t):
    """Integers as the kernels want them; what does not fit becomes the nearest that does, and is out of range there too."""
    return t if t.dtype == torch.int32 else t.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)


def _is_integer(t):
    return not t.is_floating_point() and not t.is_complex()


def _check_sizes(**sizes):
    """What goes to the library in 32 bits."""
    for name, n in sizes.items():
        assert n < 2 ** 31, f"{name} must fit 31 bits, got {n}"


def _check_cache(k_cache, v_cache, block_table, cache_lens):
    """Checks, and ``block_table`` and ``cache_lens`` as the kernels want them."""
    assert k_cache.ndim == 4 and k_cache.shape == v_cache.shape, "k_cache and v_cache must be (num_pages, page_size, nhead_k, headdim)"
    assert k_cache.dtype == v_cache.dtype and k_cache.dtype in _DTYPES, "k_cache and v_cache must share a dtype of bfloat16, float16 or float32"
    assert min(k_cache.shape) > 0, "k_cache and v_cache must not be empty"
    assert k_cache.shape[3] <= 256, "headdim above 256 is not supported"
    assert block_table.ndim == 2 and block_table.shape[1] > 0, "block_table must be (batch, max_pages)"
    assert cache_lens.shape == block_table.shape[:1], "cache_lens must have one entry per row of block_table"
    assert _is_integer(block_table) and _is_integer(cache_lens), "block_table and cache_lens must be integer tensors"
    _check_sizes(num_pages=k_cache.shape[0], page_size=k_cache.shape[1], nhead_k=k_cache.shape[2], batch=block_table.shape[0])
    assert block_table.shape[1] * k_cache.shape[1] < 2 ** 31 - 4096, "max_pages * page_size must fit 31 bits"
    block_table = _int32(block_table)
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    return block_table, _int32(cache_lens).contiguous()


def _check_writable(name, *tensors):
    """Tensors that are written in place: no element may be two."""
    for t in tensors:
        assert not any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())), f"{name}: a tensor that is written to must not be expanded"


def _cache_args(k_cache, v_cache, block_table, cache_lens):
    c = _lib.Cache()
    c.k, c.v = k_cache.data_ptr(), v_cache.data_ptr()
    for i in range(4):
        c.k_stride[i], c.v_stride[i] = k_cache.stride(i), v_cache.stride(i)
    c.block_table, c.table_stride, c.lens = block_table.data_ptr(), block_table.stride(0), cache_lens.data_ptr()
    c.num_pages, c.page_size, c.nhead_k, c.headdim = k_cache.shape
    c.batch, c.max_pages = block_table.shape
    c.dtype = _DTYPES[k_cache.dtype]
    return c


def _check_weights(key_weights, batch, nhead_k, capacity):
    assert key_weights.dtype == torch.float32 and key_weights.ndim == 3 and key_weights.stride(2) == 1, \
        "key_weights must be float32 (batch, nhead_k, positions) with unit stride along the positions"
    assert key_weights.shape[:2] == (batch, nhead_k) and key_weights.shape[2] >= capacity, \
        f"key_weights must be (batch, nhead_k, at least max_pages * page_size) = ({batch}, {nhead_k}, >= {capacity})"


def _touch(*tensors):
    """Written in place: what autograd has saved of them is no longer what it was."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _run(name, args, device):
    rc = getattr(_lib.load(), name)(ctypes.byref(args), torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {_lib.last_error()}")


def append_to_cache(k, v, cu_seqlens, k_cache, v_cache, block_table, cache_lens):
    """Writes new tokens behind those that every sequence holds already: row ``cu_seqlens[b] + i`` of ``k`` and ``v`` (packed
    ``(total, nhead_k, headdim)``, any strides) goes to position ``cache_lens[b] + i`` of sequence ``b``.  Rows outside every sequence are
    not read; a ``cu_seqlens`` that leaves ``[0, total]`` is cut to it, and ``last_status()`` says ``HBSA_STATUS_CACHE_BOUNDS``.  Returns
    the new lengths, int32 ``[batch]``; ``cache_lens`` itself is left as it is."""
    new_lens = _host.append(k, v, cu_seqlens, k_cache, v_cache, block_table, cache_lens)     # None: what it does not take goes on here
    if new_lens is not None:
        return new_lens
    _same_device(k, v, cu_seqlens, k_cache, v_cache, block_table, cache_lens)
    _refuse_gradients("append_to_cache", k, v, k_cache, v_cache)
    block_table, lens = _check_cache(k_cache, v_cache, block_table, cache_lens)
    _check_writable("append_to_cache", k_cache, v_cache)
    assert k.ndim == 3 and k.shape == v.shape and k.shape[1:] == k_cache.shape[2:], "k and v must be (total, nhead_k, headdim) like the cache's"
    assert k.dtype == v.dtype == k_cache.dtype, "k and v must have the cache's dtype"
    assert cu_seqlens.ndim == 1 and cu_seqlens.numel() == lens.numel() + 1, "cu_seqlens must be a 1D tensor of length batch + 1"
    _check_sizes(total=k.shape[0])
    cu = _int32(cu_seqlens).contiguous()
    dev = k.device
    with torch.cuda.device(dev):
        new_lens = torch.empty(lens.shape, dtype=torch.int32, device=dev)
        if lens.numel() == 0:
            return new_lens
        status = torch.empty(4 * _lib.STATUS_WORDS, dtype=torch.uint8, device=dev)
        a = _lib.AppendArgs()
        a.struct_bytes = ctypes.sizeof(a)
        a.cache = _cache_args(k_cache, v_cache, block_table, lens)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        for i in range(3):
            a.k_stride[i], a.v_stride[i] = k.stride(i), v.stride(i)
        a.cu_seqlens, a.new_lens, a.status, a.total = cu.data_ptr(), new_lens.data_ptr(), status.data_ptr(), k.shape[0]
        _run("hbsa_append_to_cache", a, dev)
        _touch(k_cache, v_cache)
        _state["last_workspace"] = status
    return new_lens


def paged_attention(q, k_cache, v_cache, block_table, cache_lens, softmax_scale=None, block_mask=None, k_block_size=None, key_weights=None,
                    return_lse=False):
    """Attention of one new token per sequence, ``q`` ``(batch, nhead_q, headdim)``, over the sequence's cache (which holds the token's own
    key and value if it is to see itself).  Returns a contiguous tensor like ``q``, zeros for sequences that see no key; with
    ``return_lse`` also the natural-log sum of exponentials of the scaled scores, float32 ``[batch, nhead_q]``, ``-inf`` where there are none.

    ``block_mask``: bool ``(batch, nhead_k, num_k_block)`` over blocks of ``k_block_size`` positions (a multiple of 16) from the start of
    every sequence; keys of blocks that are not set are left out.  It has to cover ``max_pages * page_size`` positions.
    ``key_weights``: float32 ``(batch, nhead_k, >= max_pages * page_size)``; the attention weight of every key, summed over the q-heads of
    its kv-head, is added to it in place (what ``select_keys`` chooses by).  The call then holds every score for its duration: 4 bytes per
    q-head and position of ``batch * max_pages * page_size``."""
    result = _host.paged(q, k_cache, v_cache, block_table, cache_lens, softmax_scale, block_mask, k_block_size, key_weights, bool(return_lse))
    if result is not None:
        return result
    _same_device(q, k_cache, v_cache, block_table, cache_lens, block_mask, key_weights)
    _refuse_gradients("paged_attention", q, k_cache, v_cache, key_weights)
    block_table, lens = _check_cache(k_cache, v_cache, block_table, cache_lens)
    batch, capacity = block_table.shape[0], block_table.shape[1] * k_cache.shape[1]
    nhead_k, headdim = k_cache.shape[2:]
    assert q.ndim == 3 and q.shape[0] == batch and q.shape[2] == headdim, "q must be (batch, nhead_q, headdim) with the cache's headdim"
    assert q.dtype == k_cache.dtype, "q must have the cache's dtype"
    assert q.shape[1] > 0 and q.shape[1] % nhead_k == 0, "nhead_q must be divisible by nhead_k (for GQA)"
    _check_sizes(nhead_q=q.shape[1])
    if block_mask is not None:
        assert block_mask.dtype == torch.bool, "block_mask must be a boolean tensor"
        assert k_block_size is not None and k_block_size > 0 and k_block_size % 16 == 0, "k_block_size must be an integer multiple of 16."
        assert block_mask.ndim == 3 and block_mask.shape[:2] == (batch, nhead_k) and block_mask.shape[2] * k_block_size >= capacity, \
            f"block_mask must be ({batch}, {nhead_k}, num_k_block) and cover max_pages * page_size = {capacity} positions"
        _check_sizes(k_block_size=k_block_size, num_k_block=block_mask.shape[2])
    if key_weights is not None:
        _check_weights(key_weights, batch, nhead_k, capacity)
        _check_writable("paged_attention", key_weights)
    dev = q.device
    lib = _lib.load()
    with torch.cuda.device(dev):
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if return_lse else None
        if batch > 0:
            a = _lib.PagedAttentionArgs()
            a.struct_bytes = ctypes.sizeof(a)
            a.cache = _cache_args(k_cache, v_cache, block_table, lens)
            a.q, a.o = q.data_ptr(), out.data_ptr()
            for i in range(3):
                a.q_stride[i], a.o_stride[i] = q.stride(i), out.stride(i)
            if block_mask is not None:
                a.block_mask, a.num_k_block, a.k_block_size = block_mask.data_ptr(), block_mask.shape[2], int(k_block_size)
                for i in range(3):
                    a.mask_stride[i] = block_mask.stride(i)
            if key_weights is not None:
                a.key_weights = key_weights.data_ptr()
                a.weights_stride[0], a.weights_stride[1] = key_weights.stride(0), key_weights.stride(1)
            a.lse = lse.data_ptr() if return_lse else None
            a.nhead_q = q.shape[1]
            a.use_default_scale = 1 if softmax_scale is None else 0
            a.softmax_scale = 0.0 if softmax_scale is None else float(softmax_scale)
            a.impl = _IMPLS[_state["impl"]]
            ws = torch.empty(lib.hbsa_paged_attention_workspace_bytes(ctypes.byref(a)), dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
            _run("hbsa_paged_attention", a, dev)
            _touch(key_weights)
            _state["last_workspace"] = ws
    return (out, lse) if return_lse else out


def _key_weights(q, k, lse, cu_q_seqlens, cu_k_seqlens, mask, csr, num_q_block, num_k_block, q_block_size, k_block_size, causal,
                 softmax_scale):
    assert q.shape[1] % k.shape[1] == 0, "nhead_q must be divisible by nhead_k (for GQA)"
    assert q_block_size % 16 == 0 and k_block_size % 16 == 0 and q_block_size > 0 and k_block_size > 0, \
        "q_block_size and k_block_size must be integer multiples of 16."
    assert lse.dtype == torch.float32 and lse.shape == q.shape[:2], "lse must be float32 [total_q, nhead_q]"
    _check_sizes(total_q=q.shape[0], total_k=k.shape[0], q_block_size=q_block_size, k_block_size=k_block_size, num_q_block=num_q_block,
                 num_k_block=num_k_block)
    lse = lse.contiguous()
    lib = _lib.load()
    dev = q.device
    with torch.cuda.device(dev):
        weights = torch.empty((k.shape[0], k.shape[1]), dtype=torch.float32, device=dev)
        if q.shape[0] == 0 or k.shape[0] == 0:
            return weights.zero_()
        ws = alloc_workspace(k.shape[1], num_q_block, num_k_block, cu_q_seqlens.numel() - 1, dev)
        a = _lib.KeyWeightsArgs()
        a.struct_bytes = ctypes.sizeof(a)
        a.fwd = make_args(q, k, k, None, cu_q_seqlens, cu_k_seqlens, mask, q_block_size, k_block_size, causal, softmax_scale, num_q_block,
                          num_k_block, ws, _IMPLS[_state["impl"]], lse=lse, csr=csr)
        a.weights = weights.data_ptr()
        part = torch.empty(lib.hbsa_key_weights_workspace_bytes(ctypes.byref(a)), dtype=torch.uint8, device=dev)
        a.partial_workspace, a.partial_workspace_bytes = part.data_ptr(), part.numel()
        _run("hbsa_key_weights", a, dev)
        _state["last_workspace"] = ws
    return weights


def attention_key_weights(q, k, lse, cu_q_seqlens, cu_k_seqlens, block_mask, q_block_size, k_block_size, causal, softmax_scale=None):
    """The attention weight that the queries of a ``HBSAttention`` call give to every key: float32 ``(total_k, nhead_k)``, summed over the
    rows that see the key and over the q-heads of its kv-head.  ``lse`` is what ``HBSAttention_with_lse`` has returned for the same
    arguments; rows whose ``lse`` is ``-inf`` add nothing, keys outside every sample get zeros.  The call does not wait for the device; a
    mask that contradicts the lengths gives zeros and ``last_status()`` says so, and should the kernel give up, the weights are NaN."""
    weights = _host.key_weights(q, k, lse, cu_q_seqlens, cu_k_seqlens, block_mask, q_block_size, k_block_size, causal, softmax_scale)
    if weights is not None:
        return weights
    _same_device(q, k, lse, cu_q_seqlens, cu_k_seqlens, block_mask)
    _refuse_gradients("attention_key_weights", q, k, lse)
    assert block_mask.dtype == torch.bool, "block_mask must be a boolean tensor"
    assert block_mask.ndim == 3 and block_mask.shape[0] == k.shape[1] and min(block_mask.shape) > 0, \
        f"block_mask must be a boolean tensor of shape (nheads_k, num_q_block, num_k_block); nheads_k = {k.shape[1]}"
    cu_q32, cu_k32 = _prepare(q, k, k, cu_q_seqlens, cu_k_seqlens, block_mask)
    return _key_weights(q, k, lse, cu_q32, cu_k32, block_mask, None, block_mask.shape[1], block_mask.shape[2], q_block_size,
                        k_block_size, causal, softmax_scale)


def attention_key_weights_csr(q, k, lse, cu_q_seqlens, cu_k_seqlens, csr_row_ptr, csr_col_idx, num_q_block, num_k_block, q_block_size,
                              k_block_size, causal, softmax_scale=None):
    """``attention_key_weights`` for a block mask in CSR form (see ``HBSAttention_csr``)."""
    _same_device(q, k, lse, cu_q_seqlens, cu_k_seqlens, csr_row_ptr, csr_col_idx)
    _refuse_gradients("attention_key_weights_csr", q, k, lse)
    cu_q32, cu_k32 = _prepare(q, k, k, cu_q_seqlens, cu_k_seqlens, csr_row_ptr)
    csr = _check_csr(csr_row_ptr, csr_col_idx, k.shape[1], num_q_block)
    return _key_weights(q, k, lse, cu_q32, cu_k32, None, csr, num_q_block, num_k_block, q_block_size, k_block_size, causal,
                        softmax_scale)


def select_keys(key_weights, cache_lens, budget, n_sink=0, n_recent=0):
    """Which positions of every sequence and kv-head stay when a cache is cut to ``budget`` positions: the first ``n_sink``, the last
    ``n_recent``, and of those in between the ones of the largest weight (of equal weights the lowest positions; NaN counts as the
    largest).  ``key_weights``: float32 ``(batch, nhead_k, positions)``; ``cache_lens`` are cut to its positions.  Returns ``(kept,
    kept_lens)``: int32 ``(batch, nhead_k, budget)``, ascending, ``-1`` behind the last, and int32 ``[batch]``."""
    result = _host.select(key_weights, cache_lens, budget, n_sink, n_recent)
    if result is not None:
        return result
    _same_device(key_weights, cache_lens)
    _refuse_gradients("select_keys", key_weights)
    assert key_weights.dtype == torch.float32 and key_weights.ndim == 3 and key_weights.shape[2] > 0, "key_weights must be float32 (batch, nhead_k, positions)"
    assert key_weights.shape[2] < 2 ** 31 - 16384, "the positions must fit 31 bits"
    assert cache_lens.shape == key_weights.shape[:1] and _is_integer(cache_lens), "cache_lens must be an integer tensor of length batch"
    assert budget > 0 and n_sink >= 0 and n_recent >= 0 and n_sink + n_recent <= budget, \
        "budget must be positive, n_sink and n_recent not negative and together not above budget"
    _check_sizes(budget=budget, batch=key_weights.shape[0], nhead_k=key_weights.shape[1])
    if key_weights.stride(2) != 1:
        key_weights = key_weights.contiguous()
    lens = _int32(cache_lens).contiguous()
    dev = key_weights.device
    batch, nhead_k, size = key_weights.shape
    with torch.cuda.device(dev):
        kept = torch.empty((batch, nhead_k, int(budget)), dtype=torch.int32, device=dev)
        kept_lens = torch.empty(batch, dtype=torch.int32, device=dev)
        if batch > 0 and nhead_k > 0:
            a = _lib.SelectKeysArgs()
            a.struct_bytes = ctypes.sizeof(a)
            a.key_weights, a.lens, a.kept, a.kept_lens = key_weights.data_ptr(), lens.data_ptr(), kept.data_ptr(), kept_lens.data_ptr()
            a.weights_stride[0], a.weights_stride[1] = key_weights.stride(0), key_weights.stride(1)
            a.batch, a.nhead_k, a.max_len, a.budget, a.n_sink, a.n_recent = batch, nhead_k, size, int(budget), int(n_sink), int(n_recent)
            _run("hbsa_select_keys", a, dev)
    return kept, kept_lens


def compact_cache(k_cache, v_cache, block_table, cache_lens, kept, kept_lens, key_weights=None):
    """Moves the kept positions of every sequence and kv-head to its front, in place: position ``j`` becomes what position ``kept[b, h, j]``
    was, ``j < kept_lens[b]``.  ``kept`` (int32 ``(batch, nhead_k, budget)``) has to ascend, as that of ``select_keys`` does, and a page
    must belong to one sequence only; entries outside ``[0, cache_lens[b])`` move nothing.  ``key_weights`` (as for ``paged_attention``) move
    alike, and those of the positions that have become free turn zero.  ``cache_lens`` are the lengths before the move; ``kept_lens`` are
    those after it, for the calls that follow."""
    if _host.compact(k_cache, v_cache, block_table, cache_lens, kept, kept_lens, key_weights) is not None:
        return
    _same_device(k_cache, v_cache, block_table, cache_lens, kept, kept_lens, key_weights)
    _refuse_gradients("compact_cache", k_cache, v_cache, key_weights)
    block_table, lens = _check_cache(k_cache, v_cache, block_table, cache_lens)
    _check_writable("compact_cache", k_cache, v_cache)
    batch, nhead_k = block_table.shape[0], k_cache.shape[2]
    assert kept.ndim == 3 and kept.shape[:2] == (batch, nhead_k) and kept.shape[2] > 0 and _is_integer(kept), \
        f"kept must be an integer tensor of shape (batch, nhead_k, budget) = ({batch}, {nhead_k}, ...)"
    assert kept_lens.shape == lens.shape and _is_integer(kept_lens), "kept_lens must be an integer tensor of length batch"
    _check_sizes(budget=kept.shape[2])
    if key_weights is not None:
        _check_weights(key_weights, batch, nhead_k, block_table.shape[1] * k_cache.shape[1])
        _check_writable("compact_cache", key_weights)
    kept, kept_lens = _int32(kept).contiguous(), _int32(kept_lens).contiguous()
    dev = k_cache.device
    if batch == 0:
        return
    with torch.cuda.device(dev):
        a = _lib.CompactArgs()
        a.struct_bytes = ctypes.sizeof(a)
        a.cache = _cache_args(k_cache, v_cache, block_table, lens)
        a.kept, a.kept_lens, a.budget = kept.data_ptr(), kept_lens.data_ptr(), kept.shape[2]
        if key_weights is not None:
            a.key_weights = key_weights.data_ptr()
            a.weights_stride[0], a.weights_stride[1] = key_weights.stride(0), key_weights.stride(1)
        _run("hbsa_compact_cache", a, dev)
        _touch(k_cache, v_cache, key_weights)
