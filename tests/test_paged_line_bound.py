"""Calls whose work could not be numbered in 31 bits are refused on the host (no GPU needed)."""

from test_serving_abi import BAD, attention


def test_one_sequence_past_the_bound_is_refused():
    """2^20 tokens of 2 query heads a K/V head are 2^17 tiles of 16 rows for each of two heads; behind
    2^29 keys that is 2^41 units of 64 keys."""
    long = dict(n=2 ** 20, cols=2 ** 25, ld=2 ** 25)
    assert attention(B=1, **long) == BAD
    assert attention(B=2, **long) == BAD  # in two halves, neither of which fits
    assert attention("lk_shared_prefix_attention", B=1, n=2 ** 20, cols=0, table=None, prefix_length=2 ** 29) == BAD
