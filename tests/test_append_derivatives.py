"""The append of keys and values has no derivative, and says so: inputs that one is asked of are refused
before anything else is looked at (no GPU needed)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import llm_kernels

CACHE, SLOTS = torch.zeros(2, 16, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64)


def append(k, v, q=None):
    kw = dict(q=q, positions=SLOTS, cos_sin=llm_kernels.rotary_table(4, 64, device="cpu")) if q is not None else {}
    llm_kernels.paged_kv_append(k, v, CACHE, CACHE.clone(), SLOTS, **kw)


def test_inputs_that_need_a_gradient_are_refused():
    plain = torch.zeros(3, 2, 64, dtype=torch.float16)
    need = plain.clone().requires_grad_()
    for args in ((need, plain), (plain, need), (plain, plain, need)):
        with pytest.raises(llm_kernels.LKInputError, match="no gradient"):
            append(*args)
        # Without grad mode nothing is lost: the call gets as far as its other checks.
        with torch.no_grad(), pytest.raises(llm_kernels.LKInputError, match="CUDA"):
            append(*args)
    with pytest.raises(llm_kernels.LKInputError, match="CUDA"):
        append(need.detach(), plain)


def test_tangents_are_refused():
    plain = torch.zeros(3, 2, 64, dtype=torch.float16)
    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(plain, torch.ones_like(plain))
        for args in ((dual, plain), (plain, dual), (plain, plain, dual)):
            with pytest.raises(llm_kernels.LKInputError, match="no gradient"):
                append(*args)
