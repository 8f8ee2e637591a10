"""Host-side checks of the rotary, cache and paged-attention entry points: nothing here needs a GPU."""

import pytest
import torch

import llm_kernels
from llm_kernels import _lib

BAD, UNSUPPORTED, ALIGNMENT, OK = _lib.LK_ERR_INVALID_ARG, _lib.LK_ERR_UNSUPPORTED, _lib.LK_ERR_ALIGNMENT, _lib.LK_OK


def rotary(**kw):
    a = dict(q=4096, q_out=4096, k=4096, k_out=4096, strides=_lib.i64_array([64, 64, 64] * 4), dtype=_lib.LK_BF16, B=1, S=1, H=2,
             Hk=1, D=64, pos=4096, pos_dtype=_lib.LK_I64, pos_strides=_lib.i64_array([0, 0, 1]), table=4096, rows=8, pairs=32,
             axes=1, sections=None, interleaved=0, inverse=0, stream=None)
    a.update(kw)
    return _lib.load().lk_rotary_embed(*a.values())


def test_rotary_arguments():
    for kw in (dict(B=-1), dict(q=None), dict(k_out=None), dict(strides=None), dict(table=None), dict(pos=None), dict(rows=0),
               dict(pairs=0), dict(pairs=33), dict(axes=5), dict(axes=2), dict(axes=2, sections=_lib.i64_array([16, 15])),
               dict(axes=2, sections=_lib.i64_array([33, -1])), dict(S=2 ** 31)):
        assert rotary(**kw) == BAD, kw
    assert rotary(dtype=_lib.LK_F32) == UNSUPPORTED and rotary(pos_dtype=_lib.LK_F32) == UNSUPPORTED
    assert rotary(table=4100) == ALIGNMENT
    assert rotary(B=0) == OK and rotary(H=0, Hk=0) == OK


def append(**kw):
    a = dict(q=None, q_out=None, k=4096, v=4096, kc=4096, vc=4096, strides=_lib.i64_array([64] * 14), dtype=_lib.LK_F16, T=4, H=0,
             Hk=2, D=64, pages=4, page=16, slots=4096, slots_dtype=_lib.LK_I64, pos=None, pos_dtype=0, pos_strides=None,
             table=None, rows=0, pairs=0, axes=0, sections=None, interleaved=0, stream=None)
    a.update(kw)
    return _lib.load().lk_paged_kv_append(*a.values())


def test_append_arguments():
    for kw in (dict(T=-1), dict(k=None), dict(kc=None), dict(slots=None), dict(page=0), dict(pages=-1), dict(strides=None),
               dict(H=2, q=4096, q_out=4096), dict(table=4096)):
        assert append(**kw) == BAD, kw
    assert append(dtype=_lib.LK_F32) == UNSUPPORTED and append(slots_dtype=_lib.LK_F32) == UNSUPPORTED
    assert append(T=0) == OK


def attention(name="lk_paged_attention", **kw):
    a = dict(q=4096, kc=4096, vc=4096, table=4096, ld=4, cols=4, lengths=4096, out=4096, lse=None, strides=_lib.i64_array([64] * 12),
             dtype=_lib.LK_BF16, B=2, n=1, H=4, Hk=2, D=64, pages=8, page=16, scale=0.0, ws=None, ws_bytes=0, stream=None)
    if name != "lk_paged_attention":
        a = {"q": 4096, "kc": 4096, "vc": 4096, "prefix": 4096, "prefix_length": 5, **a}
    a.update(kw)
    return getattr(_lib.load(), name)(*a.values())


def test_attention_arguments():
    for kw in (dict(B=-1), dict(q=None), dict(kc=None), dict(table=None), dict(lengths=None), dict(out=None), dict(strides=None),
               dict(Hk=3), dict(Hk=0), dict(page=0), dict(B=2 ** 20, n=2 ** 20), dict(cols=2 ** 40), dict(pages=2 ** 33)):
        assert attention(**kw) == BAD, kw
    for kw in (dict(D=60), dict(D=136), dict(D=4), dict(dtype=_lib.LK_F32)):
        assert attention(**kw) == UNSUPPORTED, kw
    assert attention(q=4104) == ALIGNMENT and attention(strides=_lib.i64_array([64] * 11 + [4])) == ALIGNMENT
    assert attention(B=0) == OK and attention(n=0) == OK
    for kw in (dict(prefix=None), dict(prefix_length=-1)):
        assert attention("lk_shared_prefix_attention", **kw) == BAD, kw


def test_workspace_grows_with_what_it_holds():
    size = _lib.load().lk_paged_attention_workspace_bytes
    assert 0 < size(1, 1, 8, 8, 64, 0) <= size(1, 1, 8, 8, 128, 0) <= size(1, 64, 8, 8, 128, 0) < size(1, 64, 8, 8, 128, 1000)
    assert size(4, 1, 8, 8, 128, 0) % 256 == 0 and size(0, 1, 8, 8, 128, 0) == 0


def test_cpu_tensors_are_refused():
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    table, one = llm_kernels.rotary_table(4, 64, device="cpu"), torch.zeros(1, dtype=torch.int32)
    cache, pages = h(2, 16, 2, 64), torch.zeros(1, 1, dtype=torch.int32)
    for call in (
        lambda: llm_kernels.rotary_embed(h(1, 2, 64), h(1, 1, 64), one, table),
        lambda: llm_kernels.paged_kv_append(h(1, 2, 64), h(1, 2, 64), cache, cache.clone(), one),
        lambda: llm_kernels.paged_attention(h(1, 4, 64), cache, cache, pages, one),
        lambda: llm_kernels.shared_prefix_attention(h(1, 4, 64), cache, cache, one, 3, pages, one),
    ):
        with pytest.raises(llm_kernels.LKInputError, match="CUDA"):
            call()
    for call in (lambda: llm_kernels.rotary_embed(None, None, one, table), lambda: llm_kernels.paged_attention(1, 2, 3, 4, 5),
                 lambda: llm_kernels.paged_kv_append("k", "v", cache, cache, one)):
        with pytest.raises(llm_kernels.LKInputError):
            call()


def test_rotary_table():
    t = llm_kernels.rotary_table(300, 64, base=500.0, device="cpu")
    assert t.shape == (300, 32, 2) and t.dtype == torch.float32
    angle = torch.arange(300, dtype=torch.float64)[:, None] * 500.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert (t[..., 0].double() - angle.cos()).abs().max() <= 2.0 ** -24 and (t[..., 1].double() - angle.sin()).abs().max() <= 2.0 ** -24
    for bad in ((0, 64), (4, 63), (4, 0)):
        with pytest.raises(llm_kernels.LKInputError):
            llm_kernels.rotary_table(*bad, device="cpu")


def test_cache_slots():
    table = torch.tensor([[5, 2, -1], [0, 7, 9]])
    got = llm_kernels.cache_slots(table, torch.tensor([3, 10]), 4, 4).view(2, 4)
    assert got.tolist() == [[23, 8, 9, 10], [38, 39, -1, -1]]
    assert llm_kernels.cache_slots(table, torch.tensor([8, -1]), 2, 4).tolist() == [-1, -1, -1, 0]
    assert llm_kernels.cache_slots(table[:, :0], torch.tensor([0, 0]), 2, 4).tolist() == [-1] * 4
