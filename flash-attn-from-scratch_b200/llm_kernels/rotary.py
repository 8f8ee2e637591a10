"""Rotary position embedding on sm_100a, for positions with one or several axes.

No counterpart in the reference (its models have no positions).  Pair ``i`` of a head's first
``2 * pairs`` values is turned by the angle of the token's position on the pair's axis; the
rotation is its own gradient with the sign of the sines changed, so the backward pass is the
same kernel.
"""

from __future__ import annotations

import types

import torch
from torch.autograd import forward_ad

from . import _lib
from ._common import require

__all__ = ["rotary_table", "rotary_embed"]

def rotary_table(max_position: int, rotary_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """The ``cos_sin`` table of :func:`rotary_embed`: ``[max_position, rotary_dim // 2, 2]`` fp32,
    (cos, sin) of ``position * base ** (-2 i / rotary_dim)``, computed in 64 bits."""
    require(isinstance(max_position, int) and max_position > 0, "max_position must be a positive int")
    require(isinstance(rotary_dim, int) and rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_dim must be even and positive")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).to(device=device, dtype=torch.float32)


def _rotate(q, k, positions, cos_sin, sections, interleaved, inverse):
    rotary = _lib.binding().rotary
    out = rotary(q, k, positions, cos_sin, sections, interleaved, inverse)
    if out is None:  # a layout that the kernel does not read
        lead = (q if q is not None else k).shape[:-2]
        q, k = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (q, k))
        if sections is None:
            positions = expand_positions(positions, lead)
        out = rotary(q, k, positions, cos_sin, sections, interleaved, inverse)
    return out


def expand_positions(positions, lead):
    if positions.shape == lead:
        return positions
    require(positions.dim() <= len(lead), "positions must have the shape of q's tokens, or one that expands to it")
    try:
        return positions.expand(lead)
    except RuntimeError:
        require(False, "positions must have the shape of q's tokens, or one that expands to it")


class RotaryFunction(torch.autograd.Function):
    """The rotation with its gradient (the inverse rotation of the outputs' gradients) and its
    forward-mode derivative (the rotation of the inputs' tangents)."""

    @staticmethod
    def forward(ctx, q, k, positions, cos_sin, sections, interleaved, inverse):
        ctx.save_for_backward(positions, cos_sin)
        ctx.save_for_forward(positions, cos_sin)
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

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        positions, cos_sin = ctx.saved_tensors
        # With grad mode on, a gradient of the tangents may be asked for.
        rotate = RotaryFunction.apply if torch.is_grad_enabled() else _rotate
        return rotate(tq, tk, positions, cos_sin, *ctx.how)


# The forward-mode level that is open, -1 without one (0, "ask the tensors", where torch keeps no such
# number).  Asked first: to unpack a tensor costs 0.35 us.
LEVEL = forward_ad if hasattr(forward_ad, "_current_level") else types.SimpleNamespace(_current_level=0)


def has_tangent(x) -> bool:
    return isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None


def rotary_embed(q, k, positions, cos_sin, *, sections=None, interleaved=False, inverse=False):
    """Rotates queries and keys by their positions, in one kernel; differentiable in q and k, in
    reverse and in forward mode.

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
    require(isinstance(q, torch.Tensor), "q and k must be tensors")
    require(isinstance(cos_sin, torch.Tensor) and not cos_sin.requires_grad, "cos_sin must be a tensor that needs no gradient")
    if sections is not None:
        sections = tuple(sections)
    dual = False
    if LEVEL._current_level >= 0:
        dual = has_tangent(q)
        if k is not None and dual != has_tangent(k):  # the function's outputs all have one, or none
            return tuple(rotary_embed(x, None, positions, cos_sin, sections=sections, interleaved=interleaved, inverse=inverse)
                         for x in (q, k))
    if dual or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
        q_out, k_out = RotaryFunction.apply(q, k, positions, cos_sin, sections, interleaved, inverse)
    else:
        q_out, k_out = _rotate(q, k, positions, cos_sin, sections, interleaved, inverse)
    return q_out if k is None else (q_out, k_out)
