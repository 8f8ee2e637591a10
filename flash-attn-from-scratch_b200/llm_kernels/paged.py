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
from ._common import require
from .rotary import LEVEL, expand_positions, has_tangent

__all__ = ["cache_slots", "paged_kv_append", "paged_attention", "shared_prefix_attention"]

_grad_enabled = torch.is_grad_enabled

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

    Not differentiable: q, k or v that a derivative is asked of (grad mode with ``requires_grad``, or a
    forward-mode tangent) are refused.  Training rotates with :func:`rotary_embed`.
    """
    try:
        asked = _grad_enabled() and (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad))
    except AttributeError:  # no tensor: refused below
        asked = False
    if asked or (LEVEL._current_level >= 0 and (has_tangent(k) or has_tangent(v) or has_tangent(q))):
        require(False, "paged_kv_append has no gradient: call it under torch.no_grad(), or rotate with rotary_embed to train")
    if sections is not None:
        sections = tuple(sections)
    append = _lib.binding().append
    got = append(k, v, k_cache, v_cache, slots, q, positions, cos_sin, sections, interleaved, q_out)
    if got is False:  # a layout that the kernel does not read
        k, v = (t if t.stride(2) == 1 else t.contiguous() for t in (k, v))
        if q is not None and q.stride(2) != 1:
            q = q.contiguous()
        if positions is not None and sections is None:
            positions = expand_positions(positions, k.shape[:1])
        got = append(k, v, k_cache, v_cache, slots.contiguous(), q, positions, cos_sin, sections, interleaved, q_out)
    return got


def _packed(t):
    """A copy whose rows start on 16 bytes."""
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _attention(q, k_cache, v_cache, prefix_pages, prefix_length, block_table, lengths, softmax_scale, out, return_lse):
    attention = _lib.binding().attention
    got = attention(q, k_cache, v_cache, prefix_pages, prefix_length, block_table, lengths, softmax_scale, out, return_lse)
    if got is None:  # a layout that the kernels do not read
        if prefix_pages is not None:
            prefix_pages = prefix_pages.contiguous()
        got = attention(_packed(q), k_cache, v_cache, prefix_pages, prefix_length, block_table.contiguous(),
                        lengths.contiguous(), softmax_scale, None, return_lse)
        if out is not None:
            out.copy_(got[0] if return_lse else got)
            got = (out, got[1]) if return_lse else out
    return got


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
    return _attention(q, k_cache, v_cache, None, 0, block_table, lengths, softmax_scale, out, return_lse)


def shared_prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_length, block_table, lengths, *, softmax_scale=None,
                            out=None, return_lse=False):
    """:func:`paged_attention` for a batch whose sequences share their first ``prefix_length``
    keys, which are read and multiplied once for all of them (each sequence reads them itself where
    that is little work, or where the page size is no multiple of 8).

    Args:
        prefix_pages : [pages] int32, the pages that hold the prefix.
        prefix_length : int, its count of keys; every query sees all of them.
        block_table, lengths : each sequence's own pages and keys after the prefix, which begin at
            the start of a page; a length may be 0.
        The others are those of :func:`paged_attention`.
    """
    require(prefix_pages is not None, "prefix_pages must be int32 [pages]")
    return _attention(q, k_cache, v_cache, prefix_pages, prefix_length, block_table, lengths, softmax_scale, out, return_lse)
