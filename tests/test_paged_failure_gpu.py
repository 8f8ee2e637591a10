"""The 256-row attention kernel's bounded waits: a page that never arrives is reported, every role
unwinds, and the next calls are right.

As in test_failure_path_gpu.py: a one-shot hook lets one TMA load of a tiny launch never complete, with
the wait limit at 20 ms; nothing faults or hangs, and the launch returns within a few limits.  What the call
leaves in its joins' counters goes with the workspaces that clear_device_status drops."""

import pytest
import torch

import llm_kernels
from llm_kernels import _lib
from test_failure_path_gpu import _expect_timeout, short_waits
from test_paged_gpu import Case

pytestmark = pytest.mark.gpu

WIDE_SITES = range(321, 330)  # csrc/paged_wide.cu WideSite


def lose(case, block, item):
    case.run()
    torch.cuda.synchronize()
    with short_waits():
        _lib.call("lk_debug_inject", _lib.LK_INJECT_PAGED_DROP_LOAD, block, item)
        case.call()
        _expect_timeout(WIDE_SITES)
    for _ in range(2):
        case.run()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block,item", [(0, 0), (0, 1), (0, 2), (1, 0), (1, 1)])
def test_lost_page_of_one_tile(D, block, item):
    """120 rows: both halves of one tile, K_0 K_1 V_0 V_1 in block 0, and K_2 V_2 in block 1, which shares
    the item and has to put zeros behind the sequence's end in V_2."""
    lose(Case([300], n=30, H=8, Hk=2, D=D), block, item)


@pytest.mark.parametrize("block,item", [(0, 0), (2, 1)])
def test_lost_page_of_two_tiles(block, item):
    """400 rows: two tiles of a pair, K_j V_j in turn."""
    lose(Case([500, 0], n=100, H=8, Hk=2), block, item)


@pytest.mark.parametrize("n", [1, 30])
def test_lost_page_of_a_prefix_pass(n):
    """The kernels behind it give up their waits, or have none, and return.  (V_0: a block has one unit at
    least, so two loads.)"""
    lose(Case([n + 5 * b for b in range(40)], n=n, H=8, Hk=2, prefix=6000), 0, 1)
