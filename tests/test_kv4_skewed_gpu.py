"""Attention over the 4-bit cache where one sequence is spread over almost all thread blocks and the others over one or
none each: rows of very different numbers of parts are joined in one launch (B200 only)."""
import pytest

import test_kv4_gpu as kv4_test

pytestmark = kv4_test.pytestmark
kernels = kv4_test.kernels


@pytest.mark.parametrize("lengths,kv_heads", [
    ([60000] + [16] * 63, 1),              # fewer rows than blocks
    ([40] * 30 + [30000] + [0, 1, 200], 4),
    ([30000] + [100] * 300, 2),            # more rows than blocks
    ([129] * 250 + [20000] + [5000], 2),
    ([128 * 15 * n for n in (1, 2, 3)] + [128 * n for n in range(14, 20)], 1),
])
@pytest.mark.parametrize("group_heads", [1, 5, 8, 9, 16, 24])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_one_long_among_many_short(kernels, lengths, kv_heads, group_heads, head_dim):
    kv4_test.run_attend(kernels, lengths, kv_heads * group_heads, kv_heads, head_dim, 64, 64, seed=group_heads)


@pytest.mark.parametrize("tiles", [8, 14, 15, 16, 17, 18, 31, 32, 33, 65])
@pytest.mark.parametrize("group_heads", [3, 12])
def test_numbers_of_parts(kernels, tiles, group_heads):
    """A single row of so many tiles has up to two parts more: both ways to join, and the numbers between."""
    kv4_test.run_attend(kernels, [128 * tiles - 5], group_heads, 1, 128, 128, 128, seed=tiles)
