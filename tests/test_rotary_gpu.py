"""Rotary embedding and the paged-cache append on the GPU against their definitions in 64 bits.

Tolerance: each rotated value is a c - b s in fp32 (error at most 3 * 2^-24 (|a| + |b|), the table
being the operator's input) rounded once to 16 bits (half an ulp: 2^-8 of the value for bf16,
2^-11 for fp16, and 2^-25 where fp16 is subnormal); values that pass through are exact."""

import math

import pytest
import torch

import llm_kernels
from llm_kernels import _lib

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def exact(x, positions, table, sections=None, interleaved=False, sign=1.0):
    """[..., H, D] in 64 bits: pair i as a complex number times (c + i s) of its axis' position."""
    pairs = table.shape[1]
    cs = torch.view_as_complex(table.double())
    if sign < 0:
        cs = cs.conj()
    if sections is None:
        ang = cs[positions.long()]
    else:
        parts, begin = [], 0
        for a, n in enumerate(sections):
            parts.append(cs[positions[a].long()][..., begin:begin + n])
            begin += n
        ang = torch.cat(parts, -1)
    y = x.double().clone()
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    z = torch.complex(y[..., first], y[..., second]) * ang.unsqueeze(-2)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def close(got, want, x, pairs):
    size = x.double().abs().amax(-1, keepdim=True)  # at least |a| and |b|
    tol = UNIT[got.dtype] * want.abs() + 6 * 2.0 ** -24 * size + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


def inputs(lead, H, Hk, D, dtype, seed=0, rows=777, pairs=None, axes=0):
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn(*lead, H, D, device="cuda", generator=g).to(dtype)
    k = torch.randn(*lead, Hk, D, device="cuda", generator=g).to(dtype)
    table = llm_kernels.rotary_table(rows, 2 * (pairs or D // 2))
    pos = torch.randint(0, rows, ((axes,) if axes else ()) + tuple(lead), device="cuda", generator=g)
    return q, k, table, pos


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,H,Hk,D,pairs", [
    ((1,), 1, 1, 64, 32), ((5,), 8, 2, 128, 64), ((2, 7), 3, 1, 64, 16), ((3,), 4, 4, 80, 40), ((131,), 7, 1, 128, 32),
    ((9,), 2, 1, 36, 18), ((4,), 2, 2, 10, 1), ((2,), 33, 5, 256, 128), ((3,), 2, 2, 96, 20),
])
def test_forward(dtype, interleaved, lead, H, Hk, D, pairs):
    q, k, table, pos = inputs(lead, H, Hk, D, dtype, pairs=pairs)
    for p in (pos, pos.int()):
        q2, k2 = llm_kernels.rotary_embed(q, k, p, table, interleaved=interleaved)
        close(q2, exact(q, pos, table, None, interleaved), q, pairs)
        close(k2, exact(k, pos, table, None, interleaved), k, pairs)
    alone = llm_kernels.rotary_embed(q, None, pos, table, interleaved=interleaved)
    assert torch.equal(alone, q2)


@pytest.mark.parametrize("sections", [(32, 32), (16, 24, 24), (1, 2, 3, 58), (64, 0), (13, 51), (64,)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(sections, interleaved):
    q, k, table, pos = inputs((2, 11), 4, 2, 128, torch.bfloat16, axes=len(sections))
    q2, k2 = llm_kernels.rotary_embed(q, k, pos, table, sections=sections, interleaved=interleaved)
    close(q2, exact(q, pos, table, sections, interleaved), q, 64)
    close(k2, exact(k, pos, table, sections, interleaved), k, 64)


def test_strides_and_broadcast_positions():
    q, k, table, _ = inputs((3, 10), 4, 2, 64, torch.float16)
    pos = torch.arange(10, device="cuda")
    want_q, want_k = (exact(t, pos.expand(3, 10), table) for t in (q, k))
    packed = torch.cat((q, k), 2)  # one projection's output, read through slices
    shifted = torch.empty(packed.numel() + 1, dtype=packed.dtype, device="cuda")[1:].view(packed.shape).copy_(packed)
    headed = packed.transpose(1, 2).contiguous().transpose(1, 2)  # [B, H, S, D] storage
    wide = torch.stack((packed, packed), -1)[..., 0]  # last dim not contiguous
    for t in (packed, shifted, headed, wide):
        q2, k2 = llm_kernels.rotary_embed(t[:, :, :4], t[:, :, 4:], pos, table)
        close(q2, want_q, q, 32)
        close(k2, want_k, k, 32)


def test_inverse_returns_and_empty():
    q, k, table, pos = inputs((40,), 4, 2, 128, torch.float16)
    q2, k2 = llm_kernels.rotary_embed(q, k, pos, table)
    back, _ = llm_kernels.rotary_embed(q2, k2, pos, table, inverse=True)
    close(back, exact(q2, pos, table, sign=-1.0), q2, 64)
    e = llm_kernels.rotary_embed(q[:0], k[:0], pos[:0], table)
    assert e[0].shape == (0, 4, 128) and e[1].shape == (0, 2, 128)


@pytest.mark.parametrize("sections", [None, (16, 8, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(sections, interleaved):
    axes = len(sections) if sections else 0
    q, k, table, pos = inputs((2, 9), 4, 2, 64, torch.bfloat16, axes=axes)
    q.requires_grad_(), k.requires_grad_()
    g = torch.Generator("cuda").manual_seed(5)
    gq, gk = (torch.randn(t.shape, device="cuda", generator=g).to(t.dtype) for t in (q, k))
    q2, k2 = llm_kernels.rotary_embed(q, k, pos, table, sections=sections, interleaved=interleaved)
    dq, dk = torch.autograd.grad((q2, k2), (q, k), (gq, gk))
    close(dq, exact(gq, pos, table, sections, interleaved, -1.0), gq, 32)
    close(dk, exact(gk, pos, table, sections, interleaved, -1.0), gk, 32)
    # Against differences of the (linear) definition: <g, f(x + d) - f(x)> = <f'(g), d>.
    d = torch.randn(q.shape, device="cuda", generator=g, dtype=torch.float64)
    left = (gq.double() * (exact(q.double() + d, pos, table, sections, interleaved)
                           - exact(q, pos, table, sections, interleaved))).sum()
    right = (dq.double() * d).sum()
    # The random rounding of dq's values: 2^-8 |dq| |d| each, added in quadrature, six sigma.
    assert abs(left - right) <= 6 * 2.0 ** -8 * (dq.double() * d).square().sum().sqrt()


def test_gradient_of_one_input_of_a_shared_head_and_again():
    q, k, table, pos = inputs((6,), 4, 1, 64, torch.float16)
    k.requires_grad_()
    q2, k2 = llm_kernels.rotary_embed(q, k.expand(6, 4, 64), pos, table)  # one head, broadcast
    assert not torch.equal(k2[:, 0], k[:, 0])
    (dk,) = torch.autograd.grad(k2.float().sum(), k)
    ones = torch.ones(6, 4, 64, device="cuda", dtype=torch.float16)
    one = llm_kernels.rotary_embed(ones, None, pos, table, inverse=True)
    assert torch.equal(dk, one.sum(1, keepdim=True))
    # The gradient of the gradient is the rotation itself.
    x = q.clone().requires_grad_()
    g = torch.randn_like(x).requires_grad_()
    y = llm_kernels.rotary_embed(x, None, pos, table)
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    (dg,) = torch.autograd.grad(dx, g, torch.ones_like(dx))
    assert torch.equal(dg, llm_kernels.rotary_embed(ones, None, pos, table))


def append_case(T, H, Hk, D, page, dtype, seed=1, head_major=False):
    g = torch.Generator("cuda").manual_seed(seed)
    qkv = torch.randn(T, H + 2 * Hk, D, device="cuda", generator=g).to(dtype)
    pages = T // page + 3
    shape = (pages, Hk, page, D) if head_major else (pages, page, Hk, D)
    caches = [torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(2)]
    if head_major:
        caches = [c.transpose(1, 2) for c in caches]
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    return qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], caches[0], caches[1], slots


def filled(cache, slots, rows):
    want = cache.double().clone()
    page = cache.shape[1]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < cache.shape[0] * page:
            want[s // page, s % page] = rows[t].double()
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,Hk,D,page,head_major", [
    (1, 4, 1, 64, 16, False), (17, 8, 8, 128, 16, True), (50, 6, 2, 80, 7, False), (33, 4, 2, 36, 1, False),
    (200, 32, 8, 128, 64, False),
])
def test_append(dtype, T, H, Hk, D, page, head_major):
    q, k, v, kc, vc, slots = append_case(T, H, Hk, D, page, dtype, head_major=head_major)
    slots[T // 2] = -1
    if T > 3:
        slots[0] = -7
    table = llm_kernels.rotary_table(500, D)
    pos = torch.randint(0, 500, (T,), device="cuda")
    pos[T // 2] = -1  # a padding token's position is not looked at for its key
    live = slots >= 0
    want_k, want_v = filled(kc, slots, exact(k, pos.clamp_min(0), table)), filled(vc, slots, v)
    size = k.double().abs().max()
    q2 = llm_kernels.paged_kv_append(k, v, kc, vc, slots.int(), q=q, positions=pos, cos_sin=table)
    close(q2[live], exact(q, pos.clamp_min(0), table)[live], q[live], D // 2)
    assert ((kc.double() - want_k).abs() <= UNIT[dtype] * want_k.abs() + 6 * 2.0 ** -24 * size + 2.0 ** -25).all()
    assert torch.equal(vc.double(), want_v)


def test_append_without_rotation_in_place_and_padding_only():
    q, k, v, kc, vc, slots = append_case(20, 4, 2, 64, 8, torch.bfloat16)
    want_k, want_v = filled(kc, slots, k), filled(vc, slots, v)
    assert llm_kernels.paged_kv_append(k, v, kc, vc, slots) is None
    assert torch.equal(kc.double(), want_k) and torch.equal(vc.double(), want_v)
    llm_kernels.paged_kv_append(-k, -v, kc, vc, torch.full_like(slots, -1))
    assert torch.equal(kc.double(), want_k) and torch.equal(vc.double(), want_v)
    llm_kernels.paged_kv_append(k[:0], v[:0], kc, vc, slots[:0])
    table = llm_kernels.rotary_table(100, 64)
    pos = torch.arange(20, device="cuda")
    want = llm_kernels.rotary_embed(q.contiguous(), None, pos, table)
    got = llm_kernels.paged_kv_append(k, v, kc, vc, slots, q=q, positions=pos, cos_sin=table, q_out=q)
    assert got is q and torch.equal(q, want)


def test_append_past_two_to_the_31_values():
    """A cache of more than 2^31 values: the last page's rows lie past a 32-bit offset."""
    page, Hk, D = 64, 8, 128
    pages = 2 ** 31 // (page * Hk * D) + 2
    kc = torch.zeros(pages, page, Hk, D, dtype=torch.float16, device="cuda")
    vc = torch.zeros(pages, page, Hk, D, dtype=torch.float16, device="cuda")
    k, v = torch.randn(2, 3, Hk, D, device="cuda").half()
    slots = torch.tensor([0, pages * page - 1, (pages - 1) * page], device="cuda")
    llm_kernels.paged_kv_append(k, v, kc, vc, slots)
    assert torch.equal(kc[-1, -1], k[1]) and torch.equal(vc[-1, 0], v[2]) and torch.equal(kc[0, 0], k[0])
    assert kc[-1, 1:-1].abs().max() == 0 and kc[0, 1:].abs().max() == 0


def test_indices_out_of_range_are_reported():
    q, k, v, kc, vc, slots = append_case(4, 2, 1, 64, 8, torch.float16)
    before = kc.clone()
    slots[:] = kc.shape[0] * 8 + torch.arange(4, device="cuda")
    llm_kernels.paged_kv_append(k, v, kc, vc, slots)
    assert llm_kernels.device_status()[:2] == (_lib.LK_ERR_INVALID_ARG, 302) and torch.equal(kc, before)
    llm_kernels.clear_device_status()
    table = llm_kernels.rotary_table(10, 64)
    got = llm_kernels.rotary_embed(q, None, torch.full((4,), 10, device="cuda"), table)
    assert llm_kernels.device_status()[:2] == (_lib.LK_ERR_INVALID_ARG, 301)
    assert torch.equal(got, llm_kernels.rotary_embed(q, None, torch.full((4,), 9, device="cuda"), table))
    llm_kernels.clear_device_status()
    assert llm_kernels.device_status() == (0, 0, 0, 0)


def test_another_stream():
    q, k, table, pos = inputs((64,), 8, 2, 128, torch.bfloat16)
    want = llm_kernels.rotary_embed(q, k, pos, table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = llm_kernels.rotary_embed(q, k, pos, table)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    q, k, table, pos = inputs((4,), 2, 1, 64, torch.float16)
    E = llm_kernels.LKInputError
    for bad in (
        lambda: llm_kernels.rotary_embed(q.float(), None, pos, table),
        lambda: llm_kernels.rotary_embed(q, k.bfloat16(), pos, table),
        lambda: llm_kernels.rotary_embed(q, k[:3], pos, table),
        lambda: llm_kernels.rotary_embed(q, k, pos.float(), table),
        lambda: llm_kernels.rotary_embed(q, k, pos[:3], table),
        lambda: llm_kernels.rotary_embed(q, k, pos, table.double()),
        lambda: llm_kernels.rotary_embed(q[..., :32], None, pos, table),
        lambda: llm_kernels.rotary_embed(q, k, pos, table[:0]),
        lambda: llm_kernels.rotary_embed(q, k, pos, table, sections=(16, 16)),
        lambda: llm_kernels.rotary_embed(q, k, pos.expand(2, 4), table, sections=(16, 15)),
        lambda: llm_kernels.rotary_embed(q, k, pos.cpu(), table),
        lambda: llm_kernels.rotary_embed(q, k, pos, table.clone().requires_grad_()),
    ):
        with pytest.raises(E):
            bad()
    _, k, v, kc, vc, slots = append_case(4, 2, 1, 64, 8, torch.float16)
    for bad in (
        lambda: llm_kernels.paged_kv_append(k, v[:3], kc, vc, slots),
        lambda: llm_kernels.paged_kv_append(k, v, kc.bfloat16(), vc, slots),
        lambda: llm_kernels.paged_kv_append(k, v, kc, vc[:-1], slots),
        lambda: llm_kernels.paged_kv_append(k, v, kc[..., ::2], vc[..., ::2], slots),
        lambda: llm_kernels.paged_kv_append(k, v, kc, vc, slots.float()),
        lambda: llm_kernels.paged_kv_append(k, v, kc, vc, slots[:3]),
        lambda: llm_kernels.paged_kv_append(k, v, kc, vc, slots, q=q),
        lambda: llm_kernels.paged_kv_append(k, v, kc, vc, slots, positions=pos),
        lambda: llm_kernels.paged_kv_append(k, v, kc, vc, slots, q=q[:3], positions=pos, cos_sin=table),
    ):
        with pytest.raises(E):
            bad()
