"""Paged and shared-prefix attention on the GPU against softmax(scale q K^T) V in 64 bits.

Tolerance, value by value, with u the unit roundoff of the 16-bit type (2^-8 bf16, 2^-11 fp16):
the output is rounded once (u |o|); the probabilities may be rounded to the type before they are
multiplied with V (u sum p|v|); the exponentials are good to 2^-13 relative and the scores'
fp32 sums to less (2^-12 sum p|v| for both, with the sums of p and p v); an fp16 probability
below 2^-14 loses up to 2^-25 of the largest (2^-25 times the keys times max|v|)."""

import math

import pytest
import torch

import llm_kernels
from llm_kernels import _lib

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    def __init__(self, lengths, n=1, H=8, Hk=2, D=128, page=16, dtype=torch.bfloat16, prefix=0, seed=0, head_major=False,
                 scale=1.0, poison=True):
        g = torch.Generator("cuda").manual_seed(seed)
        self.lengths_list, self.n, self.prefix, self.page = lengths, n, prefix, page
        B = len(lengths)
        counts = [-(-L // page) for L in lengths]
        pre = -(-prefix // page)
        total = sum(counts) + pre
        ids = torch.randperm(total + 2, device="cuda", generator=g).int()
        self.prefix_pages = ids[:pre]
        self.table = torch.full((B, max(counts + [1]) + 1), -1, dtype=torch.int32, device="cuda")
        at = pre
        for b, c in enumerate(counts):
            self.table[b, :c] = ids[at:at + c]
            at += c
        shape = (total + 2, Hk, page, D) if head_major else (total + 2, page, Hk, D)
        self.k, self.v = ((torch.randn(shape, device="cuda", generator=g)).to(dtype) for _ in range(2))
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.q = (torch.randn(B, n, H, D, device="cuda", generator=g) * scale).to(dtype)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        if poison:  # whatever lies behind a sequence's last key is not a number
            for b, L in enumerate(lengths):
                if L % page:
                    self.k[self.table[b, L // page], L % page:] = math.nan
                    self.v[self.table[b, L // page], L % page:] = math.nan
            if prefix % page:
                self.k[self.prefix_pages[-1], prefix % page:] = math.inf
                self.v[self.prefix_pages[-1], prefix % page:] = math.nan
            for i in ids[at:]:  # pages of nobody
                self.k[i], self.v[i] = math.nan, math.nan

    def rows(self, cache, pages, count):
        Hk, D = cache.shape[2:]
        return cache[pages[:-(-count // self.page)].long()].double().reshape(-1, Hk, D)[:count]

    def exact(self, scale=None):
        """(out, lse, size) with size = sum p|v|, and max|v| times the keys."""
        B, n, H, D = self.q.shape
        Hk = self.k.shape[2]
        out, size = torch.zeros(2, B, n, H, D, dtype=torch.float64, device="cuda")
        lse = torch.full((B, n, H), -math.inf, dtype=torch.float64, device="cuda")
        far = 0.0
        for b, L in enumerate(self.lengths_list):
            k = torch.cat((self.rows(self.k, self.prefix_pages, self.prefix), self.rows(self.k, self.table[b], L)))
            v = torch.cat((self.rows(self.v, self.prefix_pages, self.prefix), self.rows(self.v, self.table[b], L)))
            if not len(k):
                continue
            far = max(far, len(k) * float(v.abs().max()))
            k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
            x = torch.einsum("nhd,khd->nhk", self.q[b].double(), k) * (scale or D ** -0.5)
            end = self.prefix + (torch.arange(n, device="cuda") + L - n + 1).clamp_min(0)
            x = x.masked_fill((torch.arange(len(k), device="cuda") >= end[:, None])[:, None], -math.inf)
            lse[b] = torch.logsumexp(x, -1)
            p = (x - lse[b].unsqueeze(-1)).exp().nan_to_num(0.0)
            out[b] = torch.einsum("nhk,khd->nhd", p, v)
            size[b] = torch.einsum("nhk,khd->nhd", p, v.abs())
        return out, lse, size, far

    def call(self, **kw):
        if self.prefix:
            return llm_kernels.shared_prefix_attention(self.q, self.k, self.v, self.prefix_pages, self.prefix, self.table,
                                                       self.lengths, **kw)
        return llm_kernels.paged_attention(self.q, self.k, self.v, self.table, self.lengths, **kw)

    def check(self, got, lse=None, scale=None):
        want, want_lse, size, far = self.exact(scale)
        u = UNIT[self.q.dtype]
        tol = u * want.abs() + (u + 2.0 ** -12) * size + (2.0 ** -25 * far if u < 2.0 ** -10 else 0.0)
        assert got.shape == want.shape
        assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() - tol).max()
        if lse is not None:
            empty = want_lse == -math.inf
            assert torch.equal(lse == -math.inf, empty)
            # 2^-13 of each exponential, and 32-bit sums: of size 1 beside a logarithm
            assert ((lse.double() - want_lse)[~empty].abs() <= 2.0 ** -12 + 2.0 ** -18 * want_lse[~empty].abs()).all()

    def run(self):
        out, lse = self.call(return_lse=True)
        self.check(out, lse)
        # No row depends on anything but its inputs: a second call gives the same bits.
        again, lse2 = self.call(return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [0], [15, 16, 17], [1, 0, 300, 64, 65], [1000], [127, 128, 129, 0, 5000]])
def test_one_token(dtype, D, lengths):
    Case(lengths, D=D, dtype=dtype).run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 4), (7, 1), (8, 1), (16, 1), (17, 1), (40, 1), (12, 4), (28, 4)])
def test_head_groups(dtype, H, Hk):
    Case([70, 3, 513], H=H, Hk=Hk, dtype=dtype).run()


@pytest.mark.parametrize("D", [8, 24, 40, 72, 80, 96, 120])
@pytest.mark.parametrize("n", [1, 20])
def test_head_dims(D, n):
    Case([90, 33, 400], n=n, D=D, dtype=torch.float16).run()


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 100, 128, 256])
@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("head_major", [False, True])
def test_pages(page, n, head_major):
    Case([200, 1, 77, 600], n=n, page=page, head_major=head_major).run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,Hk", [(2, 8, 2), (3, 4, 4), (5, 8, 2), (16, 2, 2), (17, 2, 2), (64, 4, 1), (100, 8, 2), (300, 2, 1),
                                    (130, 7, 1)])
def test_several_tokens(dtype, n, H, Hk):
    """Lengths below, at and above the count of new tokens: some rows see nothing."""
    Case([n, 0, n - 1, n + 1, 2 * n + 133, 1], n=n, H=H, Hk=Hk, dtype=dtype).run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix", [1, 16, 100, 127, 128, 129, 2000])
@pytest.mark.parametrize("B,n,H,Hk", [(1, 1, 2, 2), (3, 1, 8, 2), (40, 1, 8, 2), (5, 3, 8, 1), (2, 50, 4, 2), (90, 1, 7, 1)])
def test_shared_prefix(dtype, prefix, B, n, H, Hk):
    lengths = [(37 * b + n) % 150 if b % 4 else (0 if b % 8 else n) for b in range(B)]
    Case(lengths, n=n, H=H, Hk=Hk, prefix=prefix, dtype=dtype).run()


@pytest.mark.parametrize("D,page", [(64, 16), (80, 64), (40, 24), (128, 3)])
@pytest.mark.parametrize("B", [2, 70])
def test_shared_prefix_layouts(D, page, B):
    Case([(11 * b) % 40 for b in range(B)], H=4, Hk=2, D=D, page=page, prefix=333, dtype=torch.float16, head_major=True).run()


def test_no_prefix_is_paged_attention():
    c = Case([50, 0, 7])
    a = llm_kernels.shared_prefix_attention(c.q, c.k, c.v, c.prefix_pages, 0, c.table, c.lengths)
    assert torch.equal(a, c.call())


def test_prefix_is_its_pages_in_front():
    """The same keys, once as a shared prefix and once as each sequence's own pages."""
    c = Case([30, 64, 1], prefix=64, H=16, Hk=2)
    table = torch.cat((c.prefix_pages.expand(3, -1), c.table), 1)
    own = llm_kernels.paged_attention(c.q, c.k, c.v, table, c.lengths + 64)
    c.check(own)
    c.check(c.call())


@pytest.mark.parametrize("n", [1, 33])
def test_many_sequences_and_one_long(n):
    """More sequences than blocks, and one whose keys are shared among all blocks."""
    Case([(7 * b) % 90 for b in range(500)], n=n, H=4, Hk=1, D=64).run()
    Case([40000, 3], n=n, H=4, Hk=1, D=64).run()


@pytest.mark.parametrize("n", [1, 20])
def test_large_scores(n):
    """Peaked softmax: scores of several hundred, running maxima that move often."""
    Case([700, 40], n=n, scale=60.0).run()
    c = Case([300], n=n, scale=1.0)
    out, lse = c.call(return_lse=True, softmax_scale=3.5)
    c.check(out, lse, scale=3.5)


@pytest.mark.parametrize("n", [1, 20])
def test_infinite_values(n):
    """A score of -inf is a key that is not there; the type's lowest value is a finite one."""
    c = Case([100, 50], n=n, H=2, Hk=2, dtype=torch.float16)
    c.q[..., 0] = 4.0
    low = torch.finfo(torch.float16).min
    for b, L in ((0, 100), (1, 50)):
        c.k[c.table[b, 0].long(), 3] = 0.0
        c.k[c.table[b, 0].long(), 3, :, 0] = -math.inf
        c.k[c.table[b, 1].long(), 5, :, 0] = low
    out, lse = c.call(return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("n,L,prefix", [(1, 20000, 0), (4, 300, 0), (40, 2500, 0), (8, 2500, 0), (20, 40000, 0), (1, 30, 5000), (300, 700, 0)])
def test_values_that_are_not_finite(n, L, prefix):
    """An infinite value stays one in its column, a key that is no number makes its head's rows so, and
    nothing else changes -- whichever blocks and shares they pass through."""
    c = Case([L, L // 2], n=n, H=8, Hk=2, prefix=prefix, dtype=torch.bfloat16, scale=0.3)
    clean = c.call()
    at = c.prefix_pages if prefix else c.table[0]
    c.v[at[0].long(), 5, 0, 17] = math.inf
    c.k[at[0].long(), 7, 1, 3] = math.nan
    out, lse = c.call(return_lse=True)
    hit = out if prefix else out[:1]
    assert (hit[:, :, :4, 17] == math.inf).all()
    assert hit[:, :, 4:].isnan().all() and (lse if prefix else lse[:1])[:, :, 4:].isnan().all()
    rest = torch.arange(128, device="cuda") != 17
    assert torch.equal(hit[:, :, :4][..., rest], (clean if prefix else clean[:1])[:, :, :4][..., rest])
    if not prefix:
        assert torch.equal(out[1], clean[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_whole_prompt_is_causal_flash_attention(dtype):
    """All of a prompt's tokens as its newest ones: the flash-attention forward's result, whose
    roundings are the same kind (its exponentials are good to 2^-13)."""
    c = Case([1500, 1500], n=1500, H=8, Hk=2, dtype=dtype, poison=False)
    got = c.call()
    k, v = (torch.stack([c.rows(x, c.table[b], 1500) for b in (0, 1)]).to(dtype).transpose(1, 2) for x in (c.k, c.v))
    other = llm_kernels.flash_attn_forward(c.q.transpose(1, 2), k, v, causal=True).transpose(1, 2)
    want, _, size, far = c.exact()
    u = UNIT[dtype]
    tol = 2 * (u * want.abs() + (u + 2.0 ** -12) * size + (2.0 ** -25 * far if u < 2.0 ** -10 else 0.0))
    assert ((got.double() - other.double()).abs() <= tol).all()


def test_offsets_past_32_bits():
    """Pages whose offsets pass 2^31 values and 2^32 bytes."""
    page, Hk, D = 64, 8, 128
    pages = 2 ** 31 // (page * Hk * D) + 8
    k = torch.zeros(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda")
    for n in (1, 30):
        c = Case([300, 100], n=n, H=16, Hk=Hk, page=page)
        used = c.k.shape[0]
        k[-used:], v[-used:] = c.k, c.v
        table = torch.where(c.table >= 0, c.table + (pages - used), -1)
        out = llm_kernels.paged_attention(c.q, k, v, table, c.lengths)
        c.check(out)


def test_strides_out_and_single_form():
    c = Case([40, 90], n=1, H=8, Hk=2)
    want = c.call()
    wide = torch.zeros(2, 8, 3, 128, dtype=c.q.dtype, device="cuda")
    wide[:, :, 1] = c.q[:, 0]
    got = llm_kernels.paged_attention(wide[:, :, 1], c.k, c.v, c.table, c.lengths)
    assert got.shape == (2, 8, 128) and torch.equal(got, want[:, 0])
    odd = torch.zeros(2 * 8 * 128 + 1, dtype=c.q.dtype, device="cuda")[1:].view(2, 8, 128)
    odd.copy_(c.q[:, 0])
    out = torch.empty(2, 8, 129, dtype=c.q.dtype, device="cuda")[..., :128]
    assert llm_kernels.paged_attention(odd, c.k, c.v, c.table, c.lengths, out=out) is out
    assert torch.equal(out, want[:, 0])
    out = torch.empty(8, 2, 128, dtype=c.q.dtype, device="cuda").transpose(0, 1)
    got, lse = llm_kernels.paged_attention(c.q[:, 0], c.k, c.v, c.table, c.lengths, out=out, return_lse=True)
    assert got is out and torch.equal(out, want[:, 0]) and lse.shape == (2, 8)
    table = c.table.t().contiguous().t()
    assert torch.equal(llm_kernels.paged_attention(c.q, c.k, c.v, table, torch.stack((c.lengths,) * 2, 1)[:, 0]), want)


def test_no_work():
    c = Case([5, 6])
    assert llm_kernels.paged_attention(c.q[:0], c.k, c.v, c.table[:0], c.lengths[:0]).shape == (0, 1, 8, 128)
    assert llm_kernels.paged_attention(c.q[:, :0], c.k, c.v, c.table, c.lengths).shape == (2, 0, 8, 128)
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    out, lse = llm_kernels.paged_attention(c.q, c.k, c.v, c.table[:, :0], zero, return_lse=True)
    assert out.abs().max() == 0 and (lse == -math.inf).all()


def test_bad_pages_and_lengths_are_reported():
    for n in (1, 20):
        c = Case([40, 90], n=n, poison=False)
        table = c.table.clone()
        table[0, 1] = c.k.shape[0]
        table[1, 0] = -1
        llm_kernels.paged_attention(c.q, c.k, c.v, table, c.lengths)
        assert llm_kernels.device_status()[:2] == (_lib.LK_ERR_INVALID_ARG, 311)
        llm_kernels.clear_device_status()
        c.check(c.call())  # and the next call is right again
        full = c.table[:, :3].clone().clamp_min(0)
        llm_kernels.paged_attention(c.q, c.k, c.v, full, c.lengths + 1000)
        assert llm_kernels.device_status()[:2] == (_lib.LK_ERR_INVALID_ARG, 312)
        llm_kernels.clear_device_status()
        neg = llm_kernels.paged_attention(c.q, c.k, c.v, c.table, -c.lengths)
        assert neg.abs().max() == 0


def test_streams_and_graphs():
    """Two streams at once, and a captured graph beside the stream that it was captured on."""
    cases = [Case([3000, 17, 900], seed=s, H=16, Hk=2, prefix=p) for s, p in ((1, 0), (2, 500))]
    want = [c.call() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = c.call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [c.call() for c in cases]
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    # New inputs in the same places.
    cases[0].lengths.copy_(torch.tensor([17, 2, 1], dtype=torch.int32))
    cases[0].lengths_list = [17, 2, 1]
    graph.replay()
    torch.cuda.synchronize()
    cases[0].check(out[0])


@pytest.mark.parametrize("B,n,prefix", [(40, 1, 3000), (70, 1, 9000), (6, 30, 5000)])
def test_prefix_pass_on_streams_and_in_a_graph(B, n, prefix):
    """The kernels of a long prefix, which overlap: beside another stream's, captured, replayed with
    other lengths, and called again at once."""
    cases = [Case([(17 * b + s) % 300 for b in range(B)], n=n, prefix=prefix, seed=s, H=8, Hk=2) for s in (0, 1)]
    want = [c.call(return_lse=True) for c in cases]
    for c, (o, lse) in zip(cases, want):
        c.check(o, lse)
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i][0]) for i in (0, 1) for o in got[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [c.call() for c in cases]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w[0]) for o, w in zip(out, want))
    cases[0].lengths_list = [max(0, L - 40) for L in cases[0].lengths_list]
    cases[0].lengths.copy_(torch.tensor(cases[0].lengths_list, dtype=torch.int32))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    cases[0].check(out[0])
    assert torch.equal(out[0], cases[0].call())


def test_slots_and_append_then_attend():
    """Tokens appended one by one and in pieces give what a whole cache gives."""
    g = torch.Generator("cuda").manual_seed(3)
    B, L, H, Hk, D, page = 3, 45, 4, 2, 64, 16
    k, v = (torch.randn(B, L, Hk, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    table = torch.randperm(12, device="cuda", generator=g).int()[:9].view(3, 3)
    kc, vc = (torch.full((12, page, Hk, D), math.nan, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    done = 0
    for n in (17, 1, 1, 20, 6):
        start = torch.full((B,), done, dtype=torch.int32, device="cuda")
        slots = llm_kernels.cache_slots(table, start, n, page)
        llm_kernels.paged_kv_append(k[:, done:done + n].reshape(-1, Hk, D), v[:, done:done + n].reshape(-1, Hk, D), kc, vc, slots)
        done += n
        c = Case([done] * B, n=n, H=H, Hk=Hk, D=D, page=page, seed=done)
        c.k, c.v, c.table = kc, vc, table
        c.lengths = start + n
        c.run()
    over = llm_kernels.cache_slots(table, torch.tensor([45, 47, -1], device="cuda"), 4, page).view(3, 4)
    assert (over[0] >= 0).tolist() == [True, True, True, False]
    assert (over[1] >= 0).tolist() == [True, False, False, False]
    assert (over[2] >= 0).tolist() == [False, True, True, True]


def test_refusals():
    c = Case([40, 90])
    E = llm_kernels.LKInputError
    P = llm_kernels.paged_attention
    for bad in (
        lambda: P(c.q.float(), c.k, c.v, c.table, c.lengths),
        lambda: P(c.q, c.k.half(), c.v.half(), c.table, c.lengths),
        lambda: P(c.q, c.k, c.v[:-1], c.table, c.lengths),
        lambda: P(c.q[..., :64], c.k, c.v, c.table, c.lengths),
        lambda: P(c.q[:, :, :7], c.k, c.v, c.table, c.lengths),
        lambda: P(c.q, c.k, c.v, c.table.long(), c.lengths),
        lambda: P(c.q, c.k, c.v, c.table[:1], c.lengths),
        lambda: P(c.q, c.k, c.v, c.table, c.lengths.long()),
        lambda: P(c.q, c.k, c.v, c.table, c.lengths[:1]),
        lambda: P(c.q, c.k, c.v, c.table, c.lengths.cpu()),
        lambda: P(c.q, c.k, c.v, c.table, c.lengths, softmax_scale=0.0),
        lambda: P(c.q, c.k, c.v, c.table, c.lengths, softmax_scale=math.nan),
        lambda: P(c.q, c.k, c.v, c.table, c.lengths, out=c.q[:1]),
        lambda: P(c.q[..., :60], c.k[..., :60], c.v[..., :60], c.table, c.lengths),
        lambda: P(c.q[..., 1:113], c.k[..., 1:113], c.v[..., 1:113], c.table, c.lengths),
        lambda: llm_kernels.shared_prefix_attention(c.q, c.k, c.v, c.table[0, :2], 33, c.table, c.lengths),
        lambda: llm_kernels.shared_prefix_attention(c.q, c.k, c.v, c.table[0, :2], -1, c.table, c.lengths),
        lambda: llm_kernels.shared_prefix_attention(c.q, c.k, c.v, c.table[0].long(), 3, c.table, c.lengths),
    ):
        with pytest.raises(E):
            bad()
    with pytest.raises(E):
        P(c.q, c.k[:0], c.v[:0], c.table, c.lengths)
    big = torch.zeros(1, 1, 2, 136, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(E):
        P(big, big, big, c.table[:1], c.lengths[:1])
