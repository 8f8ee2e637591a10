"""Rotary position embedding on sm_100a, for positions with one or several axes.

No counterpart in the reference (its models have no positions).  Pair ``i`` of a head's first
``2 * pairs`` values is turned by the angle of the token's position on the pair's axis; the
rotation is its own gradient with the sign of the sines changed, so the backward pass is the
same kernel.
"""

from __future__ import annotations

import torch

from . import _lib
from ._common import dtype_code, ptr, require, require_cuda, stream_for

__all__ = ["rotary_table", "rotary_embed"]

_INDEX_CODE = {torch.int32: _lib.LK_I32, torch.int64: _lib.LK_I64}


def rotary_table(max_position: int, rotary_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """The ``cos_sin`` table of :func:`rotary_embed`: ``[max_position, rotary_dim // 2, 2]`` fp32,
    (cos, sin) of ``position * base ** (-2 i / rotary_dim)``, computed in 64 bits."""
    require(isinstance(max_position, int) and max_position > 0, "max_position must be a positive int")
    require(isinstance(rotary_dim, int) and rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_dim must be even and positive")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).to(device=device, dtype=torch.float32)


def check_angles(positions, cos_sin, lead, D, sections):
    """Checks positions, table and sections for tokens of shape ``lead``; returns the arguments of
    the C entry points from ``positions`` to ``sections``, and the tensor that they point into."""
    require(isinstance(positions, torch.Tensor) and positions.dtype in _INDEX_CODE, "positions must be an int32 / int64 tensor")
    require(isinstance(cos_sin, torch.Tensor) and cos_sin.dtype == torch.float32 and cos_sin.dim() == 3
            and cos_sin.shape[2] == 2 and cos_sin.is_contiguous(), "cos_sin must be a contiguous fp32 [positions, pairs, 2] tensor")
    rows, pairs = cos_sin.shape[0], cos_sin.shape[1]
    require(rows > 0 and 0 < 2 * pairs <= D, "cos_sin turns more values than a head has, or has no row")
    if sections is None:
        axes, packed = 1, None
        if positions.shape != lead:
            require(positions.dim() <= len(lead), "positions must have the shape of q's tokens")
            try:
                positions = positions.expand(lead)
            except RuntimeError:
                require(False, "positions must have the shape of q's tokens, or one that expands to it")
        strides = (0, *positions.stride())
    else:
        axes = len(sections)
        require(1 <= axes <= 4 and all(isinstance(s, int) and s >= 0 for s in sections) and sum(sections) == pairs,
                "sections must be 1 to 4 counts of pairs whose sum is cos_sin's")
        require(positions.shape == (axes, *lead), "with sections, positions must be [axes, tokens...]")
        packed = _lib.pack_i64(*sections)
        strides = positions.stride()
    if len(lead) == 1:
        strides = (strides[0], 0, strides[1])
    return (ptr(positions), _INDEX_CODE[positions.dtype], _lib.pack_i64(*strides), ptr(cos_sin), rows, pairs, axes,
            packed), positions


def _outer(t):
    """(b, s, h) strides of a [B, S, H, D] or [S, H, D] tensor."""
    st = t.stride()
    return st[:3] if len(st) == 4 else (0, st[0], st[1])


def _rotate(q, k, positions, cos_sin, sections, interleaved, inverse):
    x = q if q is not None else k
    lead, D = x.shape[:-2], x.shape[-1]
    dev = require_cuda("rotary_embed", *[t for t in (q, k, positions, cos_sin) if t is not None])
    angles, positions = check_angles(positions, cos_sin, lead, D, sections)
    ins, outs, strides, args, heads = [], [], [], [], []
    for t in (q, k):
        if t is None:
            outs.append(None)
            heads.append(0)
            args += [None, None]
            strides += [0] * 6
            continue
        if t.stride(-1) != 1:
            t = t.contiguous()
        out = t.new_empty(t.shape)
        ins.append(t)
        outs.append(out)
        heads.append(t.shape[-2])
        args += [ptr(t), ptr(out)]
        strides += [*_outer(t), *_outer(out)]
    B, S = lead if len(lead) == 2 else (1, lead[0])
    _lib.call("lk_rotary_embed", *args, _lib.pack_i64(*strides), dtype_code(x.dtype), B, S, heads[0], heads[1], D,
              *angles, 1 if interleaved else 0, 1 if inverse else 0, stream_for(dev))
    return outs


class RotaryFunction(torch.autograd.Function):
    """The rotation with its gradient (the inverse rotation of the outputs' gradients)."""

    @staticmethod
    def forward(ctx, q, k, positions, cos_sin, sections, interleaved, inverse):
        ctx.save_for_backward(positions, cos_sin)
        ctx.how = (sections, interleaved, inverse)
        ctx.set_materialize_grads(False)
        q_out, k_out = _rotate(q, k, positions, cos_sin, sections, interleaved, inverse)
        return q_out, k_out

    @staticmethod
    def backward(ctx, gq, gk):
        positions, cos_sin = ctx.saved_tensors
        sections, interleaved, inverse = ctx.how
        gq = gq if ctx.needs_input_grad[0] else None
        gk = gk if ctx.needs_input_grad[1] else None
        if gq is not None or gk is not None:
            if torch.is_grad_enabled():  # a gradient of the gradient is asked for
                gq, gk = RotaryFunction.apply(gq, gk, positions, cos_sin, sections, interleaved, not inverse)
            else:
                gq, gk = _rotate(gq, gk, positions, cos_sin, sections, interleaved, not inverse)
        return gq, gk, None, None, None, None, None


def rotary_embed(q, k, positions, cos_sin, *, sections=None, interleaved=False, inverse=False):
    """Rotates queries and keys by their positions, in one kernel; differentiable in q and k.

    Args:
        q, k : [S, H, D] or [B, S, H, D] and [..., H_kv, D], fp16 / bf16 CUDA, any strides (rows
            that start on 16 bytes are fastest); k may be None.
        positions : int32 / int64, of the tokens' shape (or one that expands to it); with
            ``sections`` [axes, tokens...], e.g. the time, row and column of an image's patches.
        cos_sin : fp32 [rows, pairs, 2], as from :func:`rotary_table`; 2 * pairs <= D, values past
            2 * pairs pass through.  A position outside the rows is clamped and reported by
            ``device_status()``.
        sections : counts of pairs that go by each axis, in order (their sum is ``pairs``).
        interleaved : pair i is (x[2i], x[2i + 1]) instead of (x[i], x[i + pairs]).
        inverse : rotate back.

    Returns:
        (q', k') of q's and k's shapes and dtype, or q' alone when k is None.
    """
    require(isinstance(q, torch.Tensor) and q.dtype in (torch.float16, torch.bfloat16), "q must be an fp16 / bf16 tensor")
    require(q.dim() in (3, 4), "q must be [S, H, D] or [B, S, H, D]")
    if k is not None:
        require(isinstance(k, torch.Tensor) and k.dtype == q.dtype and k.dim() == q.dim() and k.shape[:-2] == q.shape[:-2]
                and k.shape[-1] == q.shape[-1], "k must have q's dtype, tokens and head dim")
    require(isinstance(cos_sin, torch.Tensor) and not cos_sin.requires_grad, "cos_sin must be a tensor that needs no gradient")
    if sections is not None:
        sections = tuple(sections)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        q_out, k_out = RotaryFunction.apply(q, k, positions, cos_sin, sections, interleaved, inverse)
    else:
        q_out, k_out = _rotate(q, k, positions, cos_sin, sections, interleaved, inverse)
    return q_out if k is None else (q_out, k_out)
