"""The decoder layer served from a paged cache, and rotary positions in front of the attention that
trains: the operators together, as a program uses them."""

import math

import pytest
import torch

import llm_kernels

pytestmark = pytest.mark.gpu

U = 2.0 ** -8  # bf16


def layer_of(d=512, heads=4, ff=1376):
    layer = llm_kernels.DecoderLayerOps(d_model=d, n_heads=heads, d_ff=ff).cuda()
    layer.init_weights(torch.Generator().manual_seed(4))
    return layer


def attention_exact(q, k, v):
    """Row i of q [n, H, D] sees the first len(k) - n + i + 1 keys; and sum p|v|."""
    n, L = q.shape[0], k.shape[0]
    x = torch.einsum("nhd,khd->nhk", q.double(), k.double()) * q.shape[-1] ** -0.5
    hidden = torch.arange(L, device=q.device)[None] >= torch.arange(L - n + 1, L + 1, device=q.device)[:, None]
    p = torch.softmax(x.masked_fill(hidden[:, None], -math.inf), -1)
    return torch.einsum("nhk,khd->nhd", p, v.double()), torch.einsum("nhk,khd->nhd", p, v.double().abs())


@pytest.mark.parametrize("prefix", [0, 150])
def test_layer_steps(prefix):
    """A prompt, single tokens and a few at once through the cache: each step's attention is that of
    the cache's contents, its projections those of the plain layer, and the cache holds the rotated
    keys of all tokens."""
    layer, B, H, D, page = layer_of(), 3, 4, 128, 16
    g = torch.Generator("cuda").manual_seed(0)
    table = llm_kernels.rotary_table(1000, D)
    pages = torch.randperm(60, device="cuda", generator=g).int()
    kc, vc = (torch.full((60, page, H, D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    block_table, shared, before = pages[:30].view(3, 10), None, 0
    if prefix:  # filled as a prompt of one sequence
        shared, before = pages[30:30 + -(-prefix // page)], prefix
        x = torch.randn(1, prefix, 512, device="cuda", generator=g).bfloat16()
        one = torch.tensor([prefix], dtype=torch.int32, device="cuda")
        layer.forward_cached(x, kc, vc, llm_kernels.cache_slots(shared[None], one - prefix, prefix, page), shared[None], one,
                             torch.arange(prefix, device="cuda")[None], table)
    keys = [[] for _ in range(B)]
    done = 0
    for T in (37, 1, 1, 4, 30, 1):
        x = torch.randn(B, T, 512, device="cuda", generator=g).bfloat16()
        pos = (before + done + torch.arange(T, device="cuda")).expand(B, T)
        start = torch.full((B,), done, dtype=torch.int32, device="cuda")
        slots = llm_kernels.cache_slots(block_table, start, T, page)
        u, mid = layer.forward_cached(x, kc, vc, slots, block_table, start + T, pos, table, prefix_pages=shared,
                                      prefix_length=before, return_intermediates=True)
        done += T
        q, k = llm_kernels.rotary_embed(mid["qkv"][:, :, 0], mid["qkv"][:, :, 1], pos, table)
        for b in range(B):
            keys[b].append(k[b])
            held = [c[block_table[b].long()].reshape(-1, H, D)[:done] for c in (kc, vc)]
            assert torch.equal(held[0], torch.cat(keys[b]))
            if prefix:
                held = [torch.cat((c[shared.long()].reshape(-1, H, D)[:before], h)) for c, h in zip((kc, vc), held)]
            want, size = attention_exact(q[b], *held)
            # The output's rounding, the probabilities' and 2^-12 of exponentials and 32-bit sums.
            assert ((mid["attn"][b].double() - want).abs() <= U * want.abs() + (U + 2.0 ** -12) * size).all()
        codes, scales = llm_kernels.quantize_symmetric(mid["attn"].reshape(B * T, 512))
        y = llm_kernels.int8_gemm_dequant_nk(codes, layer.o_proj.w_q, scales, layer.o_proj.scale_w)
        assert torch.equal(layer.up(y).view(B, T, -1), u)


def test_layer_without_rotation_is_the_plain_layer():
    """At angle zero the cached layer is the plain one: the same keys, causal."""
    layer, B, T, H, D, page = layer_of(), 2, 200, 4, 128, 64
    x = torch.randn(B, T, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    _, plain = layer(x, return_intermediates=True)
    kc, vc = (torch.zeros(8, page, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    zero = torch.zeros(B, T, dtype=torch.int64, device="cuda")
    lengths = torch.full((B,), T, dtype=torch.int32, device="cuda")
    slots = llm_kernels.cache_slots(table, lengths - T, T, page)
    _, mid = layer.forward_cached(x, kc, vc, slots, table, lengths, zero, llm_kernels.rotary_table(1, D), return_intermediates=True)
    assert torch.equal(mid["qkv"], plain["qkv"])
    # Two roundings of the probabilities and of the output, either kernel's.
    q, k, v = (plain["qkv"][:, :, i] for i in range(3))
    for b in range(B):
        want, size = attention_exact(q[b], k[b], v[b])
        assert ((mid["attn"][b].double() - plain["attn"][b].double()).abs() <= 2 * (U * want.abs() + (U + 2.0 ** -12) * size)).all()


def test_layer_step_in_a_graph():
    """A captured decode step, replayed with new inputs, does what the calls do."""
    layer, B, H, D, page = layer_of(), 4, 4, 128, 16
    g = torch.Generator("cuda").manual_seed(2)
    table = llm_kernels.rotary_table(1000, D)
    block_table = torch.randperm(40, device="cuda", generator=g).int().view(4, 10)
    caches = [torch.randn(40, page, H, D, device="cuda", generator=g).bfloat16() for _ in range(2)]
    x = torch.randn(B, 1, 512, device="cuda", generator=g).bfloat16()
    lengths = torch.tensor([1, 17, 60, 160], dtype=torch.int32, device="cuda")

    def step(kc, vc):
        slots = llm_kernels.cache_slots(block_table, lengths - 1, 1, page)
        return layer.forward_cached(x, kc, vc, slots, block_table, lengths, (lengths - 1).long()[:, None], table)

    step(*[c.clone() for c in caches])  # first calls allocate and load
    held = [c.clone() for c in caches]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*[c.clone() for c in caches])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for i in range(3):
        for h, c in zip(held, caches):
            h.copy_(c)
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        lengths.copy_(torch.randint(1, 161, (B,), device="cuda", generator=g))
        graph.replay()
        plain = [c.clone() for c in caches]
        assert torch.equal(out, step(*plain)) and all(torch.equal(h, c) for h, c in zip(held, plain))


@pytest.mark.parametrize("sections", [None, (16, 24, 24)])
def test_rotary_in_front_of_trained_attention(sections):
    """Gradients through the rotation and flash attention against autograd in 64 bits."""
    B, S, H, Hk, D = 1, 150, 4, 2, 128
    g = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(B, S, n, D, device="cuda", generator=g).bfloat16().requires_grad_() for n in (H, Hk, Hk))
    w = torch.randn(B, S, H, D, device="cuda", generator=g).bfloat16()
    table = llm_kernels.rotary_table(500, D)
    pos = torch.randint(0, 500, ((len(sections),) if sections else ()) + (B, S), device="cuda", generator=g)
    q2, k2 = llm_kernels.rotary_embed(q, k, pos, table, sections=sections)
    o = llm_kernels.flash_attn_with_grad(q2.transpose(1, 2), k2.transpose(1, 2), v.transpose(1, 2), causal=True)
    got = torch.autograd.grad(o, (q, k, v), w.transpose(1, 2))

    qd, kd, vd = (t.detach().double().requires_grad_() for t in (q, k, v))
    axis = torch.zeros(64, dtype=torch.long) if sections is None else torch.repeat_interleave(torch.arange(3), torch.tensor(sections))
    at = (pos[None] if sections is None else pos)[axis.cuda()]  # [pairs, B, S]
    cs = table.double()[at.permute(1, 2, 0), torch.arange(64, device="cuda")][:, :, None]

    def turn(x):
        a, b = x[..., :64], x[..., 64:]
        return torch.cat((a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]), -1)

    kk, vv = (t.repeat_interleave(H // Hk, 2) for t in (turn(kd), vd))
    x = torch.einsum("bihd,bjhd->bhij", turn(qd), kk) * D ** -0.5
    x = x.masked_fill(torch.ones(S, S, device="cuda").triu(1).bool(), -math.inf)
    want = torch.autograd.grad(torch.einsum("bhij,bjhd->bihd", torch.softmax(x, -1), vv), (qd, kd, vd), w.double())
    for a, b in zip(got, want):
        # bf16 roundings of the rotated inputs, of P and dS, of dQ / dK before they are turned back
        # and after: six of 2^-8 each, added in quadrature they stay within 3 x 2^-8 of the norm.
        assert (a.double() - b).norm() <= 3 * U * b.norm()
