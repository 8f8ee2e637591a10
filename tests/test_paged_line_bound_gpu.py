"""Block tables so wide that the work they allow for passes 31 bits, over sequences that are short: the
call goes by longer units, or takes the batch in halves, and gives the same results."""

import pytest
import torch

from test_paged_gpu import Case
from test_prefix_pass_gpu import widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,columns,prefix", [
    (12, 300_000, 0),    # 3.6 million keys: past 2^31 units of 16 keys, not of 64
    (12, 1_200_000, 0),  # 14.4 million: past 2^31 units of 64
    (16, 900_000, 0),    # the same for the 256-row kernel
    (16, 900_000, 300),  # and behind a shared prefix
])
def test_wide_tables(page, columns, prefix):
    c = Case([1500, 0, 1700, 1499, 1, 1501, 1600, 64], n=1500, H=16, Hk=2, D=64, page=page, prefix=prefix)
    items = 8 * 2 * (1500 * 8 // 16)
    assert items * columns * page // 16 > 2 ** 31
    widen(c, columns).run()
    torch.cuda.empty_cache()
