"""The 256-row attention kernel's bounded waits: a page that never arrives is reported, every role
unwinds, and the next calls are right.

As in test_failure_path_gpu.py: a one-shot hook withholds half of the bytes of a tiny launch's pages of K
or V, with the wait limit at 20 ms; nothing faults or hangs, and the launch returns within a few limits.
What the call leaves in its joins' counters goes with the workspaces that clear_device_status drops."""

import pytest
import torch

import llm_kernels
from llm_kernels import _lib
from test_failure_path_gpu import _expect_timeout, short_waits
from test_paged_gpu import Case

pytestmark = pytest.mark.gpu

WIDE_SITES = range(321, 330)  # csrc/paged_wide.cu WideSite


def lose(case, item):
    case.run()
    torch.cuda.synchronize()
    with short_waits():
        _lib.call("lk_debug_inject", _lib.LK_INJECT_PAGED_DROP_LOAD, 0, item)
        case.call()
        _expect_timeout(WIDE_SITES)
    for _ in range(2):
        case.run()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("length", [300, 1024])
@pytest.mark.parametrize("item", [0, 1])
def test_lost_pages_of_one_tile(D, length, item):
    """120 rows: both halves of one tile, in several blocks; with 300 keys one of them has to put zeros
    behind the sequence's end in a V that does not come."""
    lose(Case([length], n=30, H=8, Hk=2, D=D), item)


@pytest.mark.parametrize("item", [0, 1])
def test_lost_pages_of_two_tiles(item):
    """400 rows: two tiles of a pair, K_j V_j in turn."""
    lose(Case([500, 0], n=100, H=8, Hk=2), item)


@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("item", [0, 1])
def test_lost_pages_of_a_prefix_pass(n, item):
    """The kernels behind it give up their waits, or have none, and return."""
    lose(Case([n + 5 * b for b in range(40)], n=n, H=8, Hk=2, prefix=6000), item)
