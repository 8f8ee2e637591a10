"""A flag without a truth value raises its own error."""

import pytest
import torch

import llm_kernels

pytestmark = pytest.mark.gpu


class Neither:
    def __bool__(self):
        raise ZeroDivisionError("neither")


def test_flags_that_have_no_truth_value():
    q = torch.randn(4, 2, 64, device="cuda", dtype=torch.float16)
    table, pos = llm_kernels.rotary_table(4, 64), torch.arange(4, device="cuda")
    kc, vc = torch.zeros(2, 2, 16, 2, 64, device="cuda", dtype=torch.float16)
    pages, lengths = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    for call in (lambda: llm_kernels.rotary_embed(q, None, pos, table, interleaved=Neither()),
                 lambda: llm_kernels.rotary_embed(q, None, pos, table, inverse=Neither()),
                 lambda: llm_kernels.paged_kv_append(q, q, kc, vc, pos, q=q, positions=pos, cos_sin=table, interleaved=Neither()),
                 lambda: llm_kernels.paged_attention(q, kc, vc, pages, lengths, return_lse=Neither())):
        with pytest.raises(ZeroDivisionError, match="neither"):
            call()
    assert kc.abs().max() == 0
