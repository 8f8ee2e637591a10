"""A paged key/value cache on sm_100a: the append of new tokens, and the attention that reads it.

No counterpart in the reference, which keeps no cache.  A cache is two tensors
``[num_pages, page_size, H_kv, D]`` (keys and values; any strides with a contiguous last dim, so a
``[num_pages, H_kv, page_size, D]`` buffer is passed as its ``transpose(1, 2)``).  A sequence's
key ``j`` lies in row ``j % page_size`` of page ``block_table[b, j // page_size]``, which is slot
``page * page_size + row``.

One decode step of a layer::

    slots = cache_slots(block_table, lengths - n, n, page_size)     # once per step, for all layers
    q = paged_kv_append(k, v, k_cache, v_cache, slots, q=q, positions=pos, cos_sin=table)
    o = paged_attention(q.view(B, n, H, D), k_cache, v_cache, block_table, lengths)
"""

from __future__ import annotations

import torch

from . import _lib
from ._common import dtype_code, ptr, require, require_cuda, stream_for
from .rotary import _INDEX_CODE, check_angles

__all__ = ["cache_slots", "paged_kv_append", "paged_attention", "shared_prefix_attention"]

_HALF = (torch.float16, torch.bfloat16)


def _check_caches(k_cache, v_cache, dtype):
    require(isinstance(k_cache, torch.Tensor) and isinstance(v_cache, torch.Tensor) and k_cache.dim() == 4
            and k_cache.shape == v_cache.shape, "k_cache and v_cache must be [num_pages, page_size, H_kv, D], of one shape")
    require(k_cache.dtype == dtype and v_cache.dtype == dtype, "the caches must have the dtype of the tokens")
    require(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the caches' last dim must be contiguous")
    require(k_cache.shape[1] > 0, "page_size must be positive")


def cache_slots(block_table: torch.Tensor, starts: torch.Tensor, new: int, page_size: int) -> torch.Tensor:
    """Slots of each sequence's next ``new`` tokens, ``[B * new]`` int64: sequence b's keys
    ``starts[b] .. starts[b] + new - 1``.  A page that the block table does not have (past its
    columns, or a negative entry) gives -1.  Index arithmetic for a whole step, not per layer."""
    require(block_table.dim() == 2 and starts.shape == (block_table.shape[0],), "block_table must be [B, pages], starts [B]")
    require(isinstance(new, int) and new >= 0 and isinstance(page_size, int) and page_size > 0, "new must be >= 0, page_size > 0")
    at = starts.long()[:, None] + torch.arange(new, device=starts.device)
    col = at // page_size
    held = (at >= 0) & (col < block_table.shape[1])
    if block_table.shape[1] == 0:
        return torch.full((at.numel(),), -1, dtype=torch.int64, device=at.device)
    page = block_table.long().gather(1, col.clamp(0, block_table.shape[1] - 1))
    return torch.where(held & (page >= 0), page * page_size + at % page_size, -1).reshape(-1)


def paged_kv_append(k, v, k_cache, v_cache, slots, *, q=None, positions=None, cos_sin=None, sections=None,
                    interleaved=False, q_out=None):
    """Writes new keys (rotated by their positions) and values into their cache slots, and
    rotates the queries beside them, in one kernel.

    Args:
        k, v : [T, H_kv, D] fp16 / bf16 CUDA, e.g. slices of a fused projection's output.
        k_cache, v_cache : [num_pages, page_size, H_kv, D], written in place.
        slots : [T] int32 / int64, page * page_size + row; negative: a padding token, not written.
            No two tokens may name the same slot.  One past the cache is not written and is
            reported by ``device_status()``.
        q : [T, H, D] to rotate, optional.
        positions, cos_sin, sections, interleaved : as for :func:`rotary_embed`; without them the
            keys are written as they are (and q must be None).
        q_out : optional [T, H, D] for the rotated queries (q itself to rotate in place).

    Returns:
        the rotated queries, or None without q.
    """
    require(isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor) and k.dim() == 3 and k.dtype in _HALF
            and v.shape == k.shape and v.dtype == k.dtype, "k and v must be fp16 / bf16 [T, H_kv, D], of one shape and dtype")
    T, Hk, D = k.shape
    _check_caches(k_cache, v_cache, k.dtype)
    pages, page_size = k_cache.shape[0], k_cache.shape[1]
    require(k_cache.shape[2] == Hk and k_cache.shape[3] == D, "the caches' H_kv and D must be those of k")
    require(isinstance(slots, torch.Tensor) and slots.dtype in _INDEX_CODE and slots.shape == (T,), "slots must be int32 / int64 [T]")
    require((positions is None) == (cos_sin is None), "positions and cos_sin go together")
    require(q is not None or q_out is None, "q_out needs q")
    dev = require_cuda("paged_kv_append", k, v, k_cache, v_cache, slots)
    if slots.stride(0) != 1:
        slots = slots.contiguous()
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    H, q_ptr, qo_ptr, q_st, qo_st = 0, None, None, (0, 0), (0, 0)
    if q is not None:
        require(cos_sin is not None, "q is passed to be rotated: positions and cos_sin are needed")
        require(isinstance(q, torch.Tensor) and q.dim() == 3 and q.dtype == k.dtype and q.shape[0] == T and q.shape[2] == D
                and q.device == dev, "q must be [T, H, D] with k's dtype and device")
        if q_out is None:
            if q.stride(2) != 1:
                q = q.contiguous()
            q_out = q.new_empty(q.shape)
        else:
            require(isinstance(q_out, torch.Tensor) and q_out.shape == q.shape and q_out.dtype == q.dtype
                    and q_out.device == dev and q_out.stride(2) == 1 and q.stride(2) == 1,
                    "q_out must match q, both with a contiguous last dim")
        H, q_ptr, qo_ptr, q_st, qo_st = q.shape[1], ptr(q), ptr(q_out), q.stride()[:2], q_out.stride()[:2]
    angles = (None, 0, None, None, 0, 0, 0, None)
    if cos_sin is not None:
        require(isinstance(positions, torch.Tensor) and isinstance(cos_sin, torch.Tensor) and positions.device == dev
                and cos_sin.device == dev, "positions and cos_sin must be tensors on the caches' device")
        angles, positions = check_angles(positions, cos_sin, (T,), D, None if sections is None else tuple(sections))
    _lib.call("lk_paged_kv_append", q_ptr, qo_ptr, ptr(k), ptr(v), ptr(k_cache), ptr(v_cache),
              _lib.pack_i64(*q_st, *qo_st, *k.stride()[:2], *v.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3]),
              dtype_code(k.dtype), T, H, Hk, D, pages, page_size, ptr(slots), _INDEX_CODE[slots.dtype], *angles,
              1 if interleaved else 0, stream_for(dev))
    return q_out


# (device, stream) -> (bytes, tensor): the partial sums of sequences whose keys are shared among
# blocks, and the counters of their joins, which every call leaves at zero.  Calls on one stream
# follow one another, so they share it.
_workspaces: dict = {}


def _workspace(dev, stream, B, n, H, Hk, D, prefix):
    need = _lib.load().lk_paged_attention_workspace_bytes(B, n, H, Hk, D, prefix)
    if torch.cuda.is_current_stream_capturing():
        # A graph may be replayed beside this stream's other work: it keeps a workspace of its own.
        return torch.zeros(need, dtype=torch.uint8, device=dev), need
    held = _workspaces.get((dev, stream))
    if held is None or held[1] < need:
        held = torch.zeros(need, dtype=torch.uint8, device=dev), need
        _workspaces[(dev, stream)] = held
    return held


def _attention(name, q, k_cache, v_cache, prefix, block_table, lengths, softmax_scale, out, return_lse):
    require(isinstance(q, torch.Tensor) and q.dtype in _HALF and q.dim() in (3, 4), "q must be fp16 / bf16 [B, H, D] or [B, n, H, D]")
    single = q.dim() == 3
    if single:
        q = q.unsqueeze(1)
    B, n, H, D = q.shape
    _check_caches(k_cache, v_cache, q.dtype)
    pages, page_size, Hk = k_cache.shape[:3]
    require(k_cache.shape[3] == D, "the caches' D must be q's")
    require(Hk > 0 and H % Hk == 0, "H_kv must divide H")
    require(D % 8 == 0 and 8 <= D <= 128, "head dim must be a multiple of 8 up to 128")
    require(isinstance(block_table, torch.Tensor) and block_table.dtype == torch.int32 and block_table.dim() == 2
            and block_table.shape[0] == B, "block_table must be int32 [B, pages]")
    require(isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int32 and lengths.shape == (B,), "lengths must be int32 [B]")
    dev = require_cuda(name, q, k_cache, v_cache, block_table, lengths)
    ks, vs = k_cache.stride(), v_cache.stride()
    require(ks[0] % 8 == ks[1] % 8 == ks[2] % 8 == vs[0] % 8 == vs[1] % 8 == vs[2] % 8 == 0
            and k_cache.data_ptr() % 16 == 0 and v_cache.data_ptr() % 16 == 0, "the caches' rows must start on 16 bytes")
    if softmax_scale is None:
        scale = D ** -0.5
    else:
        scale = float(softmax_scale)
        require(0.0 < scale < float("inf"), "softmax_scale must be positive and finite")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        block_table = block_table.contiguous()
    if lengths.stride(0) != 1:
        lengths = lengths.contiguous()
    qs = q.stride()
    if qs[3] != 1 or qs[0] % 8 or qs[1] % 8 or qs[2] % 8 or q.data_ptr() % 16:
        q = torch.empty((B, n, H, D), dtype=q.dtype, device=dev).copy_(q)
        qs = q.stride()
    given = out
    if out is not None:
        require(isinstance(out, torch.Tensor) and out.dtype == q.dtype and out.device == dev
                and out.shape == ((B, H, D) if single else q.shape), "out must match q's shape, dtype and device")
        out = out.unsqueeze(1) if single else out
        os = out.stride()
        if os[3] != 1 or os[0] % 8 or os[1] % 8 or os[2] % 8 or out.data_ptr() % 16:
            out = None
    if out is None:
        out = q.new_empty((B, n, H, D))
    lse = torch.empty((B, n, H), dtype=torch.float32, device=dev) if return_lse else None
    if B and n and H:
        stream = stream_for(dev)
        ws, ws_bytes = _workspace(dev, stream, B, n, H, Hk, D, prefix[1] if prefix else 0)
        strides = _lib.pack_i64(*qs[:3], *out.stride()[:3], *ks[:3], *vs[:3])
        head = (ptr(q), ptr(k_cache), ptr(v_cache))
        tail = (ptr(block_table), block_table.stride(0), block_table.shape[1], ptr(lengths), ptr(out),
                ptr(lse) if return_lse else None, strides, dtype_code(q.dtype), B, n, H, Hk, D, pages, page_size, scale,
                ptr(ws), ws_bytes, stream)
        if prefix is None:
            _lib.call("lk_paged_attention", *head, *tail)
        else:
            _lib.call("lk_shared_prefix_attention", *head, ptr(prefix[0]), prefix[1], *tail)
    if single:
        out = out.squeeze(1)
        lse = lse.squeeze(1) if return_lse else None
    if given is not None and given.data_ptr() != out.data_ptr():
        given.copy_(out)
    if given is not None:
        out = given
    return (out, lse) if return_lse else out


def paged_attention(q, k_cache, v_cache, block_table, lengths, *, softmax_scale=None, out=None, return_lse=False):
    """Attention of each sequence's newest tokens to its pages of the cache.

    Args:
        q : [B, n, H, D] fp16 / bf16 CUDA, the n newest tokens of each sequence (their keys are
            in the cache already), or [B, H, D] for one.  D is a multiple of 8 up to 128.
        k_cache, v_cache : [num_pages, page_size, H_kv, D]; query head h reads head h // (H // H_kv).
        block_table : [B, pages] int32; entries past a sequence's last page are not read.
        lengths : [B] int32, keys of each sequence, the newest tokens' own among them.  Token i
            sees the keys below ``lengths[b] - n + i + 1``; one that sees none gives 0 (lse -inf).
        softmax_scale : defaults to D**-0.5.
        out : optional preallocated output of q's shape.
        return_lse : also return ``ln sum exp(scale q.k)`` of each row, fp32 [B, n, H] (or [B, H]).

    Page ids or lengths out of range are reported by ``device_status()``.  Not differentiable.
    """
    return _attention("paged_attention", q, k_cache, v_cache, None, block_table, lengths, softmax_scale, out, return_lse)


def shared_prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_length, block_table, lengths, *, softmax_scale=None,
                            out=None, return_lse=False):
    """:func:`paged_attention` for a batch whose sequences share their first ``prefix_length``
    keys, which are read and multiplied once for all of them.

    Args:
        prefix_pages : [pages] int32, the pages that hold the prefix.
        prefix_length : int, its count of keys; every query sees all of them.
        block_table, lengths : each sequence's own pages and keys after the prefix, which begin at
            the start of a page; a length may be 0.
        The others are those of :func:`paged_attention`.
    """
    require(isinstance(prefix_pages, torch.Tensor) and prefix_pages.dtype == torch.int32 and prefix_pages.dim() == 1,
            "prefix_pages must be int32 [pages]")
    require(isinstance(prefix_length, int) and 0 <= prefix_length, "prefix_length must be an int >= 0")
    require(isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4 and prefix_length <= prefix_pages.shape[0] * k_cache.shape[1],
            "prefix_pages holds fewer than prefix_length keys")
    require_cuda("shared_prefix_attention", q, prefix_pages)
    if prefix_pages.stride(0) != 1:
        prefix_pages = prefix_pages.contiguous()
    return _attention("shared_prefix_attention", q, k_cache, v_cache, (prefix_pages, prefix_length), block_table, lengths,
                      softmax_scale, out, return_lse)
