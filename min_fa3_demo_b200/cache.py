"""Attention over a key/value cache: writing it, trees of drafted tokens, what its slots received, and eviction.

The cache is two tensors ``[pages, page_size, KVH, 128]`` and a block table ``[B, width]`` (int32, on the device) that says
which pages hold a sequence, or, without a block table, ``[B, slots, KVH, 128]``.  Any strides will do as long as the 128
values of a head are adjacent: pages with k and v side by side, heads before slots, one layer of many.  ``cache_lens``
``[B]`` (int32, on the device) is the number of slots that are in use; no call changes it, so that the host never waits.

A decoding step: :func:`append_cache` writes the drafted tokens behind ``cache_lens``, :func:`forward_tree` lets them attend,
and once some are accepted the caller writes those again (their positions are the same) and adds them to ``cache_lens``.
:func:`cache_weights` adds up the attention that slots receive, :func:`evict_cache` drops those that received least.

No counterpart in the reference, which has no cache (``bindings.cpp:240-363`` take k and v whole).  Lengths and block
tables live on the device, so the kernels check them: what does not exist is left out, and ``check_last_status`` raises.
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import _cabi
from .min_fa3_op import (_INT32_MAX, _SCRATCH_KEPT, _SM100, _check, _check_device_capability, _on_device, _remember_workspace,
                         _stream_ptr, _workspace)
from .rotary import (_BF16, _INT32, _INT64, _NONE3, RotaryAxes, _are_positions, _check_heads, _check_positions, _is_rows, _like,
                     _position_strides, _rows)

__all__ = ["append_cache", "forward_tree", "cache_weights", "evict_cache"]


def _check_cache(cache: torch.Tensor, name: str) -> None:
    _check(cache.is_cuda, f"{name} must be a CUDA tensor")
    _check(cache.dtype == torch.bfloat16, f"{name} must have dtype torch.bfloat16")
    _check(cache.dim() == 4, f"{name} must have shape [pages, page_size, KVH, D]")
    _check(cache.size(3) == 128, f"{name} must have head_dim D=128")
    _check(cache.size(0) > 0 and cache.size(1) > 0 and cache.size(2) > 0, f"{name} must not be empty")
    _check(cache.stride(3) == 1 and not any(s & 7 for s in _rows(cache)) and cache.data_ptr() % 16 == 0,
           f"{name} must be 16-byte aligned, with adjacent values in a head and other strides multiples of 8")
    _check(all(n == 1 or s > 0 for n, s in zip(cache.shape, cache.stride())), f"{name} must not be expanded")


# As in min_fa3_op, a call first asks in few expressions whether everything is as it should be, and goes through the checks that say
# what is wrong only if not.  Here the same functions also collect what struct.pack wants, so that shapes, strides and addresses
# are asked for once (16 sequences, one token: forward_tree 19 us of host work without, 11 with).
def _is_int32(t: torch.Tensor, index: int, n: int) -> bool:
    return t.dtype is _INT32 and t.get_device() == index and t.dim() == 1 and t.size(0) == n and t.is_contiguous()


def _simple_cache(k, v, cache_lens, block_table, index: int, batch: int):
    """``b2a_cache`` for struct.pack, or None where something is wrong or needs a closer look."""
    ks, kst, kp = k.shape, k.stride(), k.data_ptr()
    if len(ks) != 4 or k.dtype is not _BF16 or index not in _SM100 or not _is_int32(cache_lens, index, batch):
        return None
    pages, size, heads, dim = ks
    k0, k1, k2, k3 = kst
    if v is None:
        vp = v0 = v1 = v2 = 0
    else:
        if v.dtype is not _BF16 or v.get_device() != index or v.shape != ks:
            return None
        vp, vst = v.data_ptr(), v.stride()
        v0, v1, v2, v3 = vst
        if v3 != 1 or v0 * v1 * v2 == 0:
            return None
    if (dim != 128 or k3 != 1 or (k0 | k1 | k2 | v0 | v1 | v2) & 7 or (kp | vp) & 15 or k0 * k1 * k2 * pages * size * heads == 0
            or batch == 0):
        return None
    if block_table is None:
        return (kp, vp, 0, 0, k0, k1, k2, v0, v1, v2, pages, size, heads, 1) if pages >= batch else None
    if block_table.dtype is not _INT32 or block_table.get_device() != index or block_table.dim() != 2 or size & 7:
        return None
    rows, width = block_table.shape
    t0, t1 = block_table.stride()
    if rows != batch or width == 0 or t1 != 1:
        return None
    return (kp, vp, block_table.data_ptr(), t0, k0, k1, k2, v0, v1, v2, pages, size, heads, width)


def _check_int32(t: torch.Tensor, name: str, shape, device) -> None:
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.device == device, f"{name} must be on the same CUDA device as the cache")
    _check(t.dtype == torch.int32, f"{name} must have dtype torch.int32")
    _check(tuple(t.shape) == tuple(shape), f"{name} must have shape {list(shape)}. Got {list(t.shape)}")
    _check(t.is_contiguous(), f"{name} must be contiguous")


def _check_table(block_table: Optional[torch.Tensor], k_cache: torch.Tensor, batch: int) -> None:
    if block_table is None:
        _check(k_cache.size(0) >= batch, f"a cache without block_table needs a row for each sequence. Got {k_cache.size(0)} for {batch}")
        return
    _check(block_table.is_cuda, "block_table must be a CUDA tensor")
    _check(block_table.device == k_cache.device, "block_table must be on the same CUDA device as the cache")
    _check(block_table.dtype == torch.int32, "block_table must have dtype torch.int32")
    _check(block_table.dim() == 2 and block_table.size(0) == batch and block_table.size(1) > 0,
           f"block_table must have shape [{batch}, width]. Got {list(block_table.shape)}")
    _check(block_table.size(1) == 1 or block_table.stride(1) == 1, "the rows of block_table must be contiguous")
    _check(k_cache.size(1) % 8 == 0, f"page_size must be a multiple of 8. Got {k_cache.size(1)}")


def _check_pair(k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    _check_cache(k_cache, "k_cache")
    _check_cache(v_cache, "v_cache")
    _check(k_cache.device == v_cache.device, "k_cache and v_cache must be on the same CUDA device")
    _check(k_cache.shape == v_cache.shape, "k_cache and v_cache must have the same shape")


def _tokens(t: torch.Tensor, name: str, batch: int, cu_seqlens: Optional[torch.Tensor], device) -> int:
    """Checks new tokens ``[B, n, H, 128]``, or ``[total, H, 128]`` with cu_seqlens; returns their number of dimensions."""
    dim = 4 if cu_seqlens is None else 3
    _check_heads(t, name, dim)
    _check(t.device == device, f"{name} must be on the same CUDA device as the cache")
    if dim == 4:
        _check(t.size(0) == batch, f"{name} must have the batch size of cache_lens. Got {t.size(0)} vs {batch}")
    return dim


def _check_lens(cache_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor], name: str, device) -> int:
    _check(cache_lens.dim() == 1 and cache_lens.numel() > 0, "cache_lens must have shape [B]")
    batch = cache_lens.numel()
    _check_int32(cache_lens, "cache_lens", (batch,), device)
    if cu_seqlens is not None:
        _check_int32(cu_seqlens, name, (batch + 1,), device)
    return batch


def _cache_fields(k_cache: torch.Tensor, v_cache: Optional[torch.Tensor], block_table: Optional[torch.Tensor]):
    """``b2a_cache`` for struct.pack, of a cache that has been checked."""
    pages, size, heads, _ = k_cache.shape
    at, width, step = (0, 1, 0) if block_table is None else (block_table.data_ptr(), block_table.size(1), block_table.stride(0))
    v = (0, _NONE3) if v_cache is None else (v_cache.data_ptr(), _rows(v_cache))
    return (k_cache.data_ptr(), v[0], at, step, *_rows(k_cache), *v[1], pages, size, heads, width)


def _check_append(k, v, k_cache, v_cache, cache_lens, block_table, cu_seqlens, q, positions, axes) -> None:
    _check_pair(k_cache, v_cache)
    device = k_cache.device
    batch = _check_lens(cache_lens, cu_seqlens, "cu_seqlens", device)
    _check_table(block_table, k_cache, batch)
    _tokens(k, "k", batch, cu_seqlens, device)
    _tokens(v, "v", batch, cu_seqlens, device)
    _check(k.shape == v.shape, "k and v must have the same shape")
    _check(k.size(-2) == k_cache.size(2), f"k and the cache must have the same KV head count. Got {k.size(-2)} vs {k_cache.size(2)}")
    _check((positions is None) == (axes is None), "positions and axes go together")
    _check(q is None or axes is not None, "q is turned by positions, so it needs positions and axes")
    if axes is not None:
        _check_positions(positions, axes, k.shape[:-2], device)
    if q is not None:
        _tokens(q, "q", batch, cu_seqlens, device)
        _check(q.shape[:-2] == k.shape[:-2], "q and k must have the same tokens")
    _check_device_capability(device, "min_fa3_demo_b200 append_cache")


_NO_POSITIONS = (0, 0)


def append_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lens: torch.Tensor, *,
                 block_table: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 axes: Optional[RotaryAxes] = None) -> Optional[torch.Tensor]:
    """Writes new tokens behind those that the cache holds, in place, and turns k (and q) by their positions on the way.

    k, v ``[B, n, KVH, 128]``, or ``[total, KVH, 128]`` with ``cu_seqlens`` ``[B + 1]`` (int32, on the device): token ``i`` of
    sequence ``b`` goes to slot ``cache_lens[b] + i``.  With ``axes`` and ``positions`` ``[axes, B, n]`` (``[axes, total]``)
    k is turned as :func:`rotary` turns it; q, if given, likewise, and is returned.  Packed tokens behind
    ``cu_seqlens[B]`` go nowhere, and their rows of the returned q are not written.  A token without a slot is left out
    and reported by ``check_last_status("append_cache")``.  No two tokens may be given the same slot by shared pages.
    """
    index, batch, ks = k_cache.get_device(), cache_lens.numel(), k.shape
    dim, tokens = 4 if cu_seqlens is None else 3, ks[:-2]
    fields = _simple_cache(k_cache, v_cache, cache_lens, block_table, index, batch)
    if not (fields is not None and _is_rows(k, dim, index) and _is_rows(v, dim, index) and v.shape == ks
            and ks[-2] == fields[12] and (ks[0] == batch if dim == 4 else _is_int32(cu_seqlens, index, batch + 1))
            and (positions is None if axes is None else positions is not None and _are_positions(positions, axes, tokens, index))
            and (q is None or (axes is not None and _is_rows(q, dim, index) and q.shape[:-2] == tokens))):
        _check_append(k, v, k_cache, v_cache, cache_lens, block_table, cu_seqlens, q, positions, axes)
        fields = _cache_fields(k_cache, v_cache, block_table)
    q_out = None if q is None else _like(q)
    if k.numel() == 0:
        return q_out
    device = k_cache.device
    ws = _workspace(16, device)
    turned = _NO_POSITIONS if axes is None else (axes._at, positions.data_ptr())
    args = _cabi.APPEND.pack(
        *fields, cache_lens.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(),
        k.data_ptr(), v.data_ptr(), 0 if q is None else q.data_ptr(), 0 if q is None else q_out.data_ptr(), *turned,
        *(_NONE3 if q is None else _rows(q)), *_rows(k), *_rows(v), *(_NONE3 if axes is None else _position_strides(positions)),
        axes is not None and positions.dtype is _INT64, batch, ks[1] if dim == 4 else 0, ks[0] * ks[1] if dim == 4 else ks[0],
        0 if q is None else q.size(-2), ws.data_ptr(), 16)
    with _on_device(device):
        _cabi.check(_cabi.load().b2a_cache_append(args, _stream_ptr(device)))
    _remember_workspace("append_cache", ws)
    return q_out


def _check_queries(q, batch, cu_seqlens_q, max_seqlen_q, tree_mask, k_cache) -> None:
    """Checks what forward_tree and cache_weights share."""
    device = k_cache.device
    dim = _tokens(q, "q", batch, cu_seqlens_q, device)
    heads, kvh = q.size(-2), k_cache.size(2)
    _check(heads > 0 and heads % kvh == 0,
           f"This demo requires qhead % kvhead == 0 for GQA/MQA. Got qhead={heads}, kvhead={kvh}")
    _check(heads // kvh <= 128, f"at most 128 query heads may share a KV head. Got qhead={heads}, kvhead={kvh}")
    if dim == 4:
        most, total = q.size(1), q.size(0) * q.size(1)
        _check(max_seqlen_q is None or int(max_seqlen_q) == most, f"max_seqlen_q must be q.size(1). Got {max_seqlen_q} vs {most}")
        _check(batch == 1 or most == 1 or q.stride(0) == most * q.stride(1), "q must have its sequences one behind the other")
        shape = (batch, most, most)
    else:
        _check(max_seqlen_q is not None and 0 < int(max_seqlen_q) <= _INT32_MAX, "packed q needs a positive max_seqlen_q")
        most, total = int(max_seqlen_q), q.size(0)
        shape = (total, most)
    _check(all(n == 1 or s > 0 for n, s in zip(q.shape, q.stride())), "q must not be expanded")
    if tree_mask is None:
        return
    _check(tree_mask.device == device, "tree_mask must be on the same CUDA device as the cache")
    _check(tree_mask.dtype == torch.bool, "tree_mask must have dtype torch.bool")
    if dim == 4:
        _check(tuple(tree_mask.shape) == shape, f"tree_mask must have shape {list(shape)}. Got {list(tree_mask.shape)}")
    else:
        _check(tree_mask.dim() == 2 and tree_mask.size(0) == total and tree_mask.size(1) >= most,
               f"tree_mask must have shape [{total}, max_seqlen_q or more]. Got {list(tree_mask.shape)}")
    _check(tree_mask.size(-1) == 1 or tree_mask.stride(-1) == 1, "the rows of tree_mask must be contiguous")


def _simple_queries(q, batch, cu_seqlens_q, max_seqlen_q, tree_mask, kvh, index):
    """(address of the mask, tokens, the most of a sequence, heads, strides of q and of the mask), or None where something is
    wrong or needs a closer look."""
    if q.dtype is not _BF16 or q.get_device() != index or q.data_ptr() & 15:
        return None
    qs, st = q.shape, q.stride()
    if cu_seqlens_q is None:
        if len(qs) != 4:
            return None
        seqs, most, heads, dim = qs
        s_seq, s_tok, s_head, s_dim = st
        total = seqs * most
        if seqs != batch or s_seq != most * s_tok or not (max_seqlen_q is None or max_seqlen_q == most):
            return None
    else:
        if len(qs) != 3 or type(max_seqlen_q) is not int or not 0 < max_seqlen_q <= _INT32_MAX or not _is_int32(cu_seqlens_q, index, batch + 1):
            return None
        total, heads, dim = qs
        s_tok, s_head, s_dim = st
        most = max_seqlen_q
    if dim != 128 or s_dim != 1 or (s_tok | s_head) & 7 or s_tok * s_head == 0 or heads % kvh or not 0 < heads <= 128 * kvh:
        return None
    if tree_mask is None:
        return 0, total, most, heads, s_tok, s_head, 0, 0
    if tree_mask.dtype is not torch.bool or tree_mask.get_device() != index:
        return None
    size, st = tree_mask.shape, tree_mask.stride()
    if st[-1] != 1:
        return None
    if cu_seqlens_q is None:
        return (tree_mask.data_ptr(), total, most, heads, s_tok, s_head, st[0], st[1]) if size == (batch, most, most) else None
    if len(size) != 2 or size[0] != total or size[1] < most:
        return None
    return tree_mask.data_ptr(), total, most, heads, s_tok, s_head, 0, st[0]


def _query_fields(q, max_seqlen_q, tree_mask):
    """What _simple_queries returns, of arguments that have been checked."""
    qs, st = q.shape, q.stride()
    at = 0 if tree_mask is None else tree_mask.data_ptr()
    if len(qs) == 4:
        mask = (0, 0) if tree_mask is None else tree_mask.stride()[:2]
        token = st[0] if qs[1] == 1 else st[1]
        return at, qs[0] * qs[1], qs[1], qs[2], token, st[2], *mask
    return at, qs[0], int(max_seqlen_q), qs[1], st[0], st[1], 0, 0 if tree_mask is None else tree_mask.stride(0)


def _check_forward_tree(q, k_cache, v_cache, cache_lens, block_table, cu_seqlens_q, max_seqlen_q, tree_mask) -> None:
    _check_pair(k_cache, v_cache)
    batch = _check_lens(cache_lens, cu_seqlens_q, "cu_seqlens_q", k_cache.device)
    _check_table(block_table, k_cache, batch)
    _check_queries(q, batch, cu_seqlens_q, max_seqlen_q, tree_mask, k_cache)
    _check_device_capability(k_cache.device, "min_fa3_demo_b200 forward_tree")


# The pieces' results (up to 38 MB) and evict_cache's lists have a buffer of their own, as in min_fa3_op: the workspace outlives the
# call.  The second allocation costs the host 1.5 us a call, of which sizes that are asked for once give back 0.5.
_TREE_KEPT = 13312            # b2a_tree_fwd_kept_workspace_bytes


@functools.lru_cache(maxsize=4096)
def _tree_bytes(lib, index: int, most: int, heads: int, kvh: int) -> Tuple[int, int]:
    """Bytes of the workspace that is kept, and of the buffer that is not; with that device current."""
    nbytes = lib.b2a_tree_fwd_workspace_bytes(most, heads, kvh)
    return (nbytes, 0) if nbytes <= _SCRATCH_KEPT else (_TREE_KEPT, nbytes - _TREE_KEPT)


@functools.lru_cache(maxsize=4096)
def _evict_bytes(lib, batch: int, kvh: int, budget: int, slots: int) -> Tuple[int, int]:
    nbytes = lib.b2a_cache_evict_workspace_bytes(batch, kvh, budget, slots)
    kept = nbytes if nbytes <= _SCRATCH_KEPT else lib.b2a_cache_evict_kept_workspace_bytes(batch)
    return kept, nbytes - kept


def forward_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_lens: torch.Tensor, *,
                 block_table: Optional[torch.Tensor] = None, cu_seqlens_q: Optional[torch.Tensor] = None,
                 max_seqlen_q: Optional[int] = None, tree_mask: Optional[torch.Tensor] = None, return_lse: bool = False,
                 out: Optional[torch.Tensor] = None):
    """Attention of drafted tokens, or of the next token, over the cache.

    q ``[B, n, QH, 128]``, or ``[total_q, QH, 128]`` with ``cu_seqlens_q`` ``[B + 1]`` (int32, on the device) and
    ``max_seqlen_q`` (its sequences one behind the other).  Token ``i`` of sequence ``b`` lies in slot ``cache_lens[b] + i`` already
    (:func:`append_cache`).  It sees all slots before ``cache_lens[b]`` and the new tokens ``u`` with ``tree_mask[b, i, u]`` (bool
    ``[B, n, n]``; packed ``[total_q, max_seqlen_q]``, a row for each token); without a mask those up to itself: ``n = 1`` is plain
    decoding.
    Returns out like q (contiguous) and, with ``return_lse``, the fp32 natural-log LSE ``[B, QH, n]`` (``[QH, total_q]``).  A row
    that sees nothing gives 0 and -inf.  Rows behind ``cu_seqlens_q[B]`` are not written; ``out`` (contiguous) may be given.
    Lengths that do not fit and pages that do not exist (their slots are seen by nobody) are reported by
    ``check_last_status("forward_tree")``.  Repeated calls give the same bits; the last bits can depend on the other sequences of
    the call.  As in ``forward``, probabilities are rounded to bf16 for their product with v (sums and LSE are of the unrounded ones):
    out is off by 0.0023 of its 2-norm on random inputs, of which its own rounding is 0.0017.
    """
    index, batch = k_cache.get_device(), cache_lens.numel()
    fields = _simple_cache(k_cache, v_cache, cache_lens, block_table, index, batch)
    query = fields and _simple_queries(q, batch, cu_seqlens_q, max_seqlen_q, tree_mask, fields[12], index)
    if query is None:
        _check_forward_tree(q, k_cache, v_cache, cache_lens, block_table, cu_seqlens_q, max_seqlen_q, tree_mask)
        fields, query = _cache_fields(k_cache, v_cache, block_table), _query_fields(q, max_seqlen_q, tree_mask)
    mask, total, most, heads, s_tok, s_head, m_seq, m_row = query
    device = k_cache.device
    if out is None:
        out = _like(q)
    else:
        _check(out.device == device and out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous(),
               "out must be contiguous and have the shape, dtype and device of q")
    if cu_seqlens_q is None:
        cu, lse = 0, torch.empty_strided((batch, heads, most), (heads * most, most, 1), dtype=torch.float32, device=device)
    else:
        cu, lse = cu_seqlens_q.data_ptr(), torch.empty_strided((heads, total), (total, 1), dtype=torch.float32, device=device)
    if total == 0:
        return (out, lse) if return_lse else out
    lib = _cabi.load()
    with _on_device(device):
        nbytes, more = _tree_bytes(lib, index, most, heads, fields[12])
        ws = _workspace(nbytes, device)
        args = _cabi.TREE.pack(*fields, cache_lens.data_ptr(), cu, q.data_ptr(), mask, out.data_ptr(), lse.data_ptr(), s_tok, s_head,
                               m_seq, m_row, batch, most, total, heads, 0.0, 0, 0, 0, 0, ws.data_ptr(), nbytes)
        if more:
            scratch = ws.new_empty(more)
            _cabi.check(lib.b2a_tree_fwd_with_scratch(args, scratch.data_ptr(), more, _stream_ptr(device)))
        else:
            _cabi.check(lib.b2a_tree_fwd(args, _stream_ptr(device)))
    _remember_workspace("forward_tree", ws)
    return (out, lse) if return_lse else out


def _check_weights(weights: torch.Tensor, batch: int, k_cache: torch.Tensor) -> None:
    kvh = k_cache.size(2)
    _check(weights.device == k_cache.device, "weights must be on the same CUDA device as the cache")
    _check(weights.dtype == torch.float32, "weights must have dtype torch.float32")
    _check(weights.dim() == 3 and weights.size(0) == batch and weights.size(1) == kvh and weights.size(2) > 0,
           f"weights must have shape [{batch}, {kvh}, slots]. Got {list(weights.shape)}")
    _check(weights.size(2) == 1 or weights.stride(2) == 1, "the rows of weights must be contiguous")


def _are_weights(weights: torch.Tensor, batch: int, kvh: int, index: int) -> bool:
    size, st = weights.shape, weights.stride()
    return (weights.dtype is torch.float32 and weights.get_device() == index and len(size) == 3 and size[0] == batch
            and size[1] == kvh and size[2] > 0 and st[2] == 1 and st[0] * st[1] > 0)


def _check_cache_weights(q, k_cache, cache_lens, weights, block_table, cu_seqlens_q, max_seqlen_q, tree_mask) -> None:
    _check_cache(k_cache, "k_cache")
    batch = _check_lens(cache_lens, cu_seqlens_q, "cu_seqlens_q", k_cache.device)
    _check_table(block_table, k_cache, batch)
    _check_queries(q, batch, cu_seqlens_q, max_seqlen_q, tree_mask, k_cache)
    _check_weights(weights, batch, k_cache)
    _check(all(n == 1 or s > 0 for n, s in zip(weights.shape, weights.stride())), "weights must not be expanded")
    _check_device_capability(k_cache.device, "min_fa3_demo_b200 cache_weights")


_WEIGHTS_WORKSPACE = 1024     # b2a_cache_weights_workspace_bytes


def cache_weights(q: torch.Tensor, lse: torch.Tensor, k_cache: torch.Tensor, cache_lens: torch.Tensor, weights: torch.Tensor, *,
                  block_table: Optional[torch.Tensor] = None, cu_seqlens_q: Optional[torch.Tensor] = None,
                  max_seqlen_q: Optional[int] = None, tree_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adds to ``weights`` ``[B, KVH, slots]`` (fp32), in place, the attention that each slot received, and returns it.

    ``weights[b, h, s]`` grows by the sum of ``exp(q k / sqrt(128) - lse)`` over the rows of K/V head ``h`` that see slot ``s``; the
    other arguments, and which slots a row sees, are those of the :func:`forward_tree` call that returned ``lse``.  Rows
    whose lse is infinite add nothing: to leave out drafted tokens that were not accepted, set theirs to infinity.  Slots behind a
    sequence are left as they were.  What does not fit is reported by ``check_last_status("cache_weights")``.
    """
    index, batch = k_cache.get_device(), cache_lens.numel()
    fields = _simple_cache(k_cache, None, cache_lens, block_table, index, batch)
    query = fields and _simple_queries(q, batch, cu_seqlens_q, max_seqlen_q, tree_mask, fields[12], index)
    if query is None or not _are_weights(weights, batch, fields[12], index):
        _check_cache_weights(q, k_cache, cache_lens, weights, block_table, cu_seqlens_q, max_seqlen_q, tree_mask)
        fields, query = _cache_fields(k_cache, None, block_table), _query_fields(q, max_seqlen_q, tree_mask)
    mask, total, most, heads, s_tok, s_head, m_seq, m_row = query
    shape, cu = ((batch, heads, most), 0) if cu_seqlens_q is None else ((heads, total), cu_seqlens_q.data_ptr())
    if not (lse.get_device() == index and lse.dtype is torch.float32 and lse.is_contiguous() and lse.shape == shape):
        raise RuntimeError(f"lse must be a contiguous torch.float32 tensor of shape {list(shape)} on the same CUDA device as the cache")
    if total == 0:
        return weights
    device = k_cache.device
    lib = _cabi.load()
    w_seq, w_head, _ = weights.stride()
    with _on_device(device):
        ws = _workspace(_WEIGHTS_WORKSPACE, device)
        args = _cabi.TREE.pack(*fields, cache_lens.data_ptr(), cu, q.data_ptr(), mask, 0, lse.data_ptr(), s_tok, s_head, m_seq, m_row,
                               batch, most, total, heads, 0.0, weights.data_ptr(), w_seq, w_head, weights.size(2), ws.data_ptr(),
                               _WEIGHTS_WORKSPACE)
        _cabi.check(lib.b2a_cache_weights(args, _stream_ptr(device)))
    _remember_workspace("cache_weights", ws)
    return weights


def _check_evict(k_cache, v_cache, weights, cache_lens, budget, recent, block_table) -> None:
    _check_pair(k_cache, v_cache)
    batch = _check_lens(cache_lens, None, "", k_cache.device)
    _check_table(block_table, k_cache, batch)
    _check_weights(weights, batch, k_cache)
    _check(0 < budget <= _INT32_MAX, f"budget must be positive. Got {budget}")
    _check(0 <= recent <= budget, f"recent must be between 0 and the budget. Got {recent}")
    _check(batch * k_cache.size(2) <= 65535, f"at most 65535 sequences times KV heads. Got {batch} times {k_cache.size(2)}")
    _check_device_capability(k_cache.device, "min_fa3_demo_b200 evict_cache")


def evict_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, cache_lens: torch.Tensor, budget: int, *,
                recent: int = 0, block_table: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts sequences longer than ``budget`` slots down to it, in place, each K/V head by itself.

    The last ``recent`` slots stay, and of the others the ``budget - recent`` with the largest ``weights`` ``[B, KVH, slots]`` (equal
    ones: the lower slot; NaN counts as largest).  Returns ``(lens, weights, index)``: the new ``cache_lens`` ``[B]``, the
    weights in the new order (0 behind the new length), and for each slot the slot that its contents come from,
    ``[B, KVH, budget]`` (int32, -1 behind the new length), for whatever else the caller keeps by slot.  Heavy slots below
    ``budget - recent`` keep their place, the gaps are filled in ascending order with the heavy ones from behind, and the last
    ones follow in their order.  Give ``weights`` no more slots than the longest sequence may have: where ``slots - budget +
    recent`` is at most 512 one launch does it all.  Sequences within the budget stay as they are.  Pages must not be shared
    between sequences.  Lengths and pages that do not exist are reported by ``check_last_status("evict_cache")``.
    """
    budget, recent = int(budget), int(recent)
    index, batch = k_cache.get_device(), cache_lens.numel()
    fields = _simple_cache(k_cache, v_cache, cache_lens, block_table, index, batch)
    if not (fields is not None and _are_weights(weights, batch, fields[12], index) and 0 <= recent <= budget <= _INT32_MAX
            and budget > 0 and batch * fields[12] <= 65535):
        _check_evict(k_cache, v_cache, weights, cache_lens, budget, recent, block_table)
        fields = _cache_fields(k_cache, v_cache, block_table)
    kvh, device, slots = fields[12], k_cache.device, weights.size(2)
    lens = torch.empty_like(cache_lens)
    new_weights = _like(weights)
    order = torch.empty_strided((batch, kvh, budget), (kvh * budget, budget, 1), dtype=_INT32, device=device)
    lib = _cabi.load()
    w_seq, w_head, _ = weights.stride()
    with _on_device(device):
        nbytes, more = _evict_bytes(lib, batch, kvh, budget, slots)
        ws = _workspace(nbytes, device)
        args = _cabi.EVICT.pack(*fields, cache_lens.data_ptr(), weights.data_ptr(), w_seq, w_head, batch, slots, budget, recent,
                                lens.data_ptr(), new_weights.data_ptr(), order.data_ptr(), ws.data_ptr(), nbytes)
        if more:
            scratch = ws.new_empty(more)
            _cabi.check(lib.b2a_cache_evict_with_scratch(args, scratch.data_ptr(), more, _stream_ptr(device)))
        else:
            _cabi.check(lib.b2a_cache_evict(args, _stream_ptr(device)))
    _remember_workspace("evict_cache", ws)
    return lens, new_weights, order
