"""The pass over a shared prefix, in all the forms that it and the pass over the own keys beside it
take.  Each case asks the workspace whether the pass ran, so that a changed rule cannot turn it into
a test of the one-kernel path.

Tolerances are those of Case.check (test_paged_gpu.py), derived there from the roundings that either
path makes."""

import math

import pytest
import torch

import llm_kernels
from llm_kernels import _lib
from test_paged_gpu import Case

pytestmark = pytest.mark.gpu

COUNTERS = 4096  # ints at the workspace's start; the last one is the pass's count of blocks


def native(c, workspace=None):
    """The C entry point on the case's tensors: (out, lse, blocks of the prefix pass or 0)."""
    B, n, H, D = c.q.shape
    num_pages, page, Hk = c.k.shape[:3]
    need = _lib.load().lk_paged_attention_workspace_bytes(B, n, H, Hk, D, c.prefix)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda") if workspace is None else workspace
    out, lse = torch.empty_like(c.q), torch.empty(B, n, H, dtype=torch.float32, device="cuda")
    strides = [*c.q.stride()[:3], *out.stride()[:3], *c.k.stride()[:3], *c.v.stride()[:3]]
    _lib.set_device(0)
    _lib.call("lk_shared_prefix_attention", c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.prefix_pages.data_ptr(), c.prefix,
              c.table.data_ptr(), c.table.stride(0), c.table.shape[1], c.lengths.data_ptr(), out.data_ptr(), lse.data_ptr(),
              _lib.i64_array(strides), _lib.LK_BF16 if c.q.dtype == torch.bfloat16 else _lib.LK_F16, B, n, H, Hk, D, num_pages,
              page, 0.0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    ints = ws[: 4 * COUNTERS].view(torch.int32).tolist()
    assert not any(ints[:-1])  # every call leaves the joins' counters at zero
    return out, lse, ints[-1]


def widen(c, pages):
    """The same case with a block table of `pages` columns, as wide as a server's longest context."""
    table = torch.full((c.table.shape[0], pages), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    c.table = table
    return c


def check(c):
    out, lse, blocks = native(c)
    assert blocks, "the prefix pass did not run"
    c.check(out, lse)
    again, lse2 = c.call(return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def lengths_of(B, n, most):
    """Empty ones, ones shorter than the new tokens, and longer ones."""
    return [0 if b % 7 == 3 else (n - 1 if b % 5 == 2 else n + (37 * b) % most) for b in range(B)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,n,H,Hk,prefix", [
    (4, 300, 8, 2, 1000),   # many rows behind a medium prefix
    (1, 500, 8, 2, 2000),   # one prompt's piece: nothing but its own tiles share the prefix
    (2, 250, 8, 2, 1000),
    (8, 8, 32, 8, 2000),    # 32 rows: two tiles of 16
])
def test_many_rows_take_the_pass(dtype, B, n, H, Hk, prefix):
    check(Case(lengths_of(B, n, 100), n=n, H=H, Hk=Hk, prefix=prefix, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page,head_major", [(128, 16, False), (64, 16, False), (64, 64, True), (40, 24, False), (80, 8, True),
                                               (128, 128, False), (120, 40, True)])
@pytest.mark.parametrize("B,n,H,Hk,prefix", [
    (32, 1, 32, 8, 1100),  # 128 rows in all: one tile, whose halves take every second block
    (90, 1, 14, 2, 2100),  # 630 rows
    (20, 30, 8, 2, 1000),  # 120 rows a sequence: their own keys take the 256-row kernel too
])
def test_forms_of_the_pass(dtype, D, page, head_major, B, n, H, Hk, prefix):
    check(Case(lengths_of(B, n, 200), n=n, H=H, Hk=Hk, D=D, page=page, prefix=prefix, dtype=dtype, head_major=head_major))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("wide_table", [False, True])
@pytest.mark.parametrize("n", [5, 8])
def test_two_tiles_of_rows(D, wide_table, n):
    """17 to 32 rows a sequence: their own keys go by the block table's width to either kernel."""
    c = Case(lengths_of(40, n, 300), n=n, H=8, Hk=2, D=D, prefix=3000)
    check(widen(c, 512) if wide_table else c)


@pytest.mark.parametrize("prefix", [500, 1000, 3001])
def test_row_tiles_on_one_line(prefix):
    """As many pairs of row tiles as would leave SMs idle side by side: all items form one line."""
    check(Case(lengths_of(19, 50, 60), n=50, H=8, Hk=1, D=64, prefix=prefix))


@pytest.mark.parametrize("prefix", [127, 128, 129, 1023, 1025, 2048])
def test_ends_of_the_prefix(prefix):
    check(Case(lengths_of(60, 40, 50), n=40, H=16, Hk=8, prefix=prefix))


@pytest.mark.parametrize("B,n,prefix", [(40, 1, 9000), (20, 30, 3000), (32, 1, 5000)])
def test_values_that_are_not_finite_behind_a_long_prefix(B, n, prefix):
    """An infinite value stays one in its column, a key that is no number makes its head's rows so, and
    nothing else changes -- through the shares of the pass and those of the own keys."""
    c = Case([n + (17 * b) % 90 for b in range(B)], n=n, H=8, Hk=2, prefix=prefix, scale=0.3)
    clean, _, blocks = native(c)
    assert blocks
    rest = torch.arange(128, device="cuda") != 17
    at, own = c.prefix_pages[3].long(), c.table[1, 0].long()
    saved = c.k[own].clone(), c.v[own].clone()
    c.v[own, 0, 0, 17] = math.inf  # a key of sequence 1 that all its tokens see
    c.k[own, 0, 1, 3] = math.nan
    out, lse, _ = native(c)
    assert (out[1, :, :4, 17] == math.inf).all() and out[1, :, 4:].isnan().all() and lse[1, :, 4:].isnan().all()
    assert torch.equal(out[1, :, :4][..., rest], clean[1, :, :4][..., rest])
    others = torch.arange(B, device="cuda") != 1
    assert torch.equal(out[others], clean[others])
    c.k[own], c.v[own] = saved
    c.v[at, 5, 0, 17] = math.inf
    c.k[at, 7, 1, 3] = math.nan
    out, lse, _ = native(c)
    assert (out[:, :, :4, 17] == math.inf).all() and out[:, :, 4:].isnan().all() and lse[:, :, 4:].isnan().all()
    assert torch.equal(out[:, :, :4][..., rest], clean[:, :, :4][..., rest])


def test_one_workspace_for_calls_of_all_forms():
    """Calls of either path on one stream share a workspace."""
    cases = [Case(lengths_of(B, n, 80), n=n, H=8, Hk=2, prefix=prefix, seed=i)
             for i, (B, n, prefix) in enumerate([(40, 1, 5000), (3, 1, 100), (20, 30, 2000), (5, 20, 64), (40, 5, 2000)])]
    size = max(_lib.load().lk_paged_attention_workspace_bytes(c.q.shape[0], c.n, 8, 2, 128, c.prefix) for c in cases)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    want = [native(c)[:2] for c in cases]
    for _ in range(3):
        for c, (out, lse) in zip(cases, want):
            got = native(c, ws)
            assert torch.equal(got[0], out) and torch.equal(got[1], lse)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 5, 8])
def test_the_pass_yields_where_the_16_row_kernel_runs_beside_it(D, n):
    """It leaves SMs to that kernel and to no other: up to 32 rows a sequence, where the block table is
    narrow, and with a wide table (where the 256-row kernel takes the own keys) to none.  The own keys are
    work enough for the pass to keep only half of its blocks."""
    case = lambda: Case([1000] * 40, n=n, H=8, Hk=2, D=D, prefix=3000)  # noqa: E731
    narrow, wide = native(case())[2], native(widen(case(), 512))[2]
    assert narrow and wide
    assert abs(narrow) < abs(wide) if n > 4 else narrow == wide


@pytest.mark.parametrize("length", [33, 2 ** 31, 2 ** 63 - 1, 2 ** 63, 2 ** 70])
def test_prefix_lengths_past_the_pages_are_refused(length):
    c = Case([5, 9], prefix=32)
    with pytest.raises(llm_kernels.LKInputError):
        llm_kernels.shared_prefix_attention(c.q, c.k, c.v, c.prefix_pages, length, c.table, c.lengths)
