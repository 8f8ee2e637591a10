"""Forward-mode derivatives of the rotation through the kernel."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import llm_kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,pairs", [(64, 32), (36, 18)])
def test_forward_mode(D, pairs):
    """The tangents of the outputs are the rotated tangents of the inputs."""
    g = torch.Generator("cuda").manual_seed(0)
    q, k, tq, tk = (torch.randn(7, n, D, device="cuda", generator=g).bfloat16() for n in (4, 2, 4, 2))
    table, pos = llm_kernels.rotary_table(50, 2 * pairs), torch.randint(0, 50, (7,), device="cuda", generator=g)
    want_q, want_k = llm_kernels.rotary_embed(tq, tk, pos, table)
    with fwd.dual_level():
        q2, k2 = llm_kernels.rotary_embed(fwd.make_dual(q, tq), fwd.make_dual(k, tk), pos, table)
        assert torch.equal(fwd.unpack_dual(q2).tangent, want_q) and torch.equal(fwd.unpack_dual(k2).tangent, want_k)
        q2, k2 = llm_kernels.rotary_embed(fwd.make_dual(q, tq), k, pos, table)
        assert torch.equal(fwd.unpack_dual(q2).tangent, want_q) and fwd.unpack_dual(k2).tangent is None
