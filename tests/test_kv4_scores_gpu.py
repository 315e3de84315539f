"""Attention over the 4-bit cache where scores are so large that FP32 holds them in whole steps (B200 only)."""
import pytest
import torch

import kv4_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


def case(kernels, lengths, seed):
    table, pages, _ = ref.scattered_table(lengths, 16, 1, seed)
    cache = ref.filled_cache(kernels, pages, 1, 16, 128, 64, seed)
    q = torch.randn((len(lengths), 8, 128), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).abs().to(BF16)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)


def set_keys(cache, table, b, first, second):
    """Keys of one value for each half of the channels, one pair of values a position."""
    for t in range(len(first)):
        cache.k_scales[table[b, t // 16].long(), 0, t % 16] = torch.tensor([[0.0, first[t]], [0.0, second[t]]], dtype=BF16, device=DEV)


@pytest.mark.parametrize("power", [10, 17, 19, 20, 21])
@pytest.mark.parametrize("loud", [0, 20])
def test_staircase(kernels, power, loud):
    """Scores near -2^(power + 6) that rise from tile to tile by some eight in the logarithm, which is what the
    reference point allows before it follows: what comes out lies between the smallest and the largest value."""
    lengths = [128 * 12, 700]
    q, cache, table, lens = case(kernels, lengths, power)
    cache.v_scales.mul_(2.0 ** loud)
    sums = q[..., 64:].double().sum(-1).mean().item()
    for step in (7.0, 8.0, 8.5, 9.0, 9.5, 10.0, 12.0, 16.0):
        for b, n in enumerate(lengths):
            set_keys(cache, table, b, [-2.0 ** power] * n, [step * 0.6931 / sums * (t // 16 % 2 + t // 32) for t in range(n)])
        out = kernels.kv4_decode(q, cache, table, lens, 1.0).double()
        for b, n in enumerate(lengths):
            pages = table[b, : -(-n // 16)].long()
            v = ref.values(cache.v_codes[pages, 0].flatten(0, 1)[:n], cache.v_scales[pages, 0].flatten(0, 1)[:n])
            size = v.abs().amax(0) * 2.0 ** -7
            assert out[b].isfinite().all()
            assert ((out[b] >= v.amin(0) - size) & (out[b] <= v.amax(0) + size)).all()
    assert kernels.device_status() == 0


@pytest.mark.parametrize("size", [1e3, 1e5, 1e6, 2e6, -1e3, -1e6, -2e6])
@pytest.mark.parametrize("place", [0, 150, 499])
def test_one_position_outweighs_all(kernels, size, place):
    """All scores some -100 size, one of them by an eighth of that higher: its value comes out, rounded.  (A weight
    times its scale is rounded by 2^-11 of at most 15 scales, the result by 2^-8.)"""
    lengths = [500]
    q, cache, table, lens = case(kernels, lengths, 7)
    keys = [-size] * 500
    keys[place] = -size + abs(size) / 8
    set_keys(cache, table, 0, keys, keys)
    out = kernels.kv4_decode(q, cache, table, lens, 1.0).double()
    at = (table[0, place // 16].long(), 0, place % 16)
    v = ref.values(cache.v_codes[at], cache.v_scales[at])
    slack = 2.0 ** -11 * 16 * cache.v_scales[at].double().abs().amax() + 2.0 ** -18 * v.abs()
    assert ((out[0] - v).abs() <= slack + 2.0 ** -8 * (v.abs() + slack)).all()


@pytest.mark.parametrize("size", [1e4, 1e6, 1e7, 1e9, 1e15, 1e30])
@pytest.mark.parametrize("first", [16, 128, 400])
def test_keys_that_weigh_nothing(kernels, size, first):
    """The first keys hold a large negative number, as a program may write them for positions that shall not count."""
    lengths = [600, 401]
    q, cache, table, lens = case(kernels, lengths, 8)
    for b in range(2):
        cache.k_scales[table[b, : first // 16].long(), 0] = torch.tensor([0.0, -size], dtype=BF16, device=DEV)
    out = kernels.kv4_decode(q, cache, table, lens, 128 ** -0.5)
    want, _, bound = ref.attend(q, cache, table[:, first // 16:], [n - first for n in lengths], 128 ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()


def test_steps_of_two(kernels):
    """Scores near -2^24 / ln 2, where FP32 counts in twos: the first tile's, then eight more in the logarithm of two,
    over values of scale 1 and zero 0, whose products with the weights come closest to FP16's largest number."""
    lengths = [128 * 40]
    q, cache, table, lens = case(kernels, lengths, 9)
    # a hundred sequences over the same pages: several tiles to a thread block
    q, table, lens = torch.ones((100, 8, 128), dtype=BF16, device=DEV), table.repeat(100, 1), lens.repeat(100)
    cache.v_scales[..., 0], cache.v_scales[..., 1] = 1.0, 0.0
    for first in range(16):
        for rise in (0.0766, 0.0864, 0.0962, 0.1064, 0.1162):
            set_keys_of_tiles(cache, table, -2.0 ** 18 * (1 + first / 128), [0.0] * 20 + [rise] * 20)
            out = kernels.kv4_decode(q, cache, table, lens, 1.0)
            assert out.isfinite().all() and (out >= 0).all() and (out <= 15).all() and (out > 0.5).any()
    assert kernels.device_status() == 0


def set_keys_of_tiles(cache, table, first, second):
    """As ``set_keys``, one value of the second half for each tile of 128 positions (eight pages)."""
    pages = table[0].long().view(len(second), 8)
    values = torch.tensor(second, dtype=BF16, device=DEV)
    cache.k_scales.zero_()
    cache.k_scales[..., 0, 1] = first
    cache.k_scales[pages, 0, :, 1, 1] = values[:, None, None]
