"""Forward-mode derivatives of the rotation, without a GPU: the Python layer over a stand-in for the
extension, which rotates in plain torch as the kernel does."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import llm_kernels
from llm_kernels import _lib


def turn(x, positions, table, sections, interleaved, inverse):
    """A plain rotation (one axis, halves)."""
    assert sections is None and not interleaved
    pairs = table.shape[1]
    cos, sin = (table[positions.long()][..., i].unsqueeze(-2).double() for i in (0, 1))
    sin = -sin if inverse else sin
    a, b, rest = x[..., :pairs].double(), x[..., pairs:2 * pairs].double(), x[..., 2 * pairs:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest.double()), -1).to(x.dtype)


class Stand:
    calls = 0

    def rotary(self, q, k, *how):
        Stand.calls += 1
        with torch.no_grad():
            return tuple(None if x is None else turn(x.detach(), *how) for x in (q, k))


@pytest.fixture(autouse=True)
def stand(monkeypatch):
    monkeypatch.setattr(_lib, "binding", lambda: Stand())


def inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, tq, tk = (torch.randn(5, n, 16, generator=g, dtype=torch.float64) for n in (3, 2, 3, 2))
    return q, k, tq, tk, torch.arange(5), llm_kernels.rotary_table(8, 12, device="cpu")


@pytest.mark.parametrize("inverse", [False, True])
def test_tangents_are_rotated(inverse):
    q, k, tq, tk, pos, table = inputs()
    want_q, want_k = (turn(t, pos, table, None, False, inverse) for t in (tq, tk))
    with fwd.dual_level():
        q2, k2 = llm_kernels.rotary_embed(fwd.make_dual(q, tq), fwd.make_dual(k, tk), pos, table, inverse=inverse)
        (q2, dq), (k2, dk) = fwd.unpack_dual(q2), fwd.unpack_dual(k2)
    assert torch.equal(dq, want_q) and torch.equal(dk, want_k)
    assert torch.equal(q2, turn(q, pos, table, None, False, inverse)) and torch.equal(k2, turn(k, pos, table, None, False, inverse))


def test_one_input_with_a_tangent_and_no_grad_mode():
    q, k, tq, tk, pos, table = inputs(1)
    with fwd.dual_level(), torch.no_grad():
        q2, k2 = llm_kernels.rotary_embed(q, fwd.make_dual(k, tk), pos, table)
        assert fwd.unpack_dual(q2).tangent is None and torch.equal(q2, turn(q, pos, table, None, False, False))
        assert torch.equal(fwd.unpack_dual(k2).tangent, turn(tk, pos, table, None, False, False))
        alone = llm_kernels.rotary_embed(fwd.make_dual(q, tq), None, pos, table)
        assert torch.equal(fwd.unpack_dual(alone).tangent, turn(tq, pos, table, None, False, False))


def test_gradient_of_a_tangent():
    """Reverse over forward: the tangent q' = R t has the gradient R^T g in t."""
    q, _, tq, _, pos, table = inputs(2)
    tq.requires_grad_()
    with fwd.dual_level():
        out = llm_kernels.rotary_embed(fwd.make_dual(q, tq), None, pos, table)
        tangent = fwd.unpack_dual(out).tangent
    (g,) = torch.autograd.grad(tangent, tq, torch.ones_like(tangent))
    assert torch.equal(g, turn(torch.ones_like(tq), pos, table, None, False, True))


def test_both_modes_at_once_and_neither():
    q, _, tq, _, pos, table = inputs(3)
    q.requires_grad_()
    with fwd.dual_level():
        out = llm_kernels.rotary_embed(fwd.make_dual(q, tq), None, pos, table)
        assert torch.equal(fwd.unpack_dual(out).tangent, turn(tq, pos, table, None, False, False))
        (g,) = torch.autograd.grad(fwd.unpack_dual(out).primal.sum(), q)
    assert torch.equal(g, turn(torch.ones_like(tq), pos, table, None, False, True))
    Stand.calls = 0
    with fwd.dual_level():  # no input has a tangent: one plain call
        out = llm_kernels.rotary_embed(q.detach(), None, pos, table)
        assert fwd.unpack_dual(out).tangent is None and Stand.calls == 1
