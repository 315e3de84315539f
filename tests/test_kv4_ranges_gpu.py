"""Attention over the 4-bit cache where value magnitudes differ within a sequence, or are very large or very
small (B200 only)."""
import math

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


def attend(q, cache, table, lengths, scale):
    """out and the bound of its error in 64 bits.

    As ``kv4_reference.attend``, but for the products of weight and scale that are smaller than FP16's normal
    numbers.  A reference point is set 2^27 below the largest product of weight and magnitude (of the
    scales and zeros of a position, taken at most twice too large, and as 2^-60 at least), the products enter
    times 2^-20, and the smallest step there is 2^-24: half a step is 2^-25 + 20 - 27 + 1 = 2^-31 of the
    largest product, and a code is at most 8 away from 8: 2^-28 for each position.  An exponential that
    is smaller than 2^-126 relative to the reference point is lost: it weighs less than 2^-126 - 27 + 1 = 2^-152
    of the largest product, above and below the line."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    group = q.shape[1] // cache.kv_heads
    for b, length in enumerate(lengths):
        pages = table[b, : -(-length // cache.page)].long()
        for h in range(cache.kv_heads):
            rows = lambda t: t[pages, h].flatten(0, 1)[:length]
            k, v = ref.values(rows(cache.k_codes), rows(cache.k_scales)), ref.values(rows(cache.v_codes), rows(cache.v_scales))
            heads = slice(h * group, (h + 1) * group)
            qh = q[b, heads].double()
            scores = qh @ k.T * scale
            pairs = rows(cache.k_scales).double()
            # a score's error by the magnitudes of its own position
            size = (15 * pairs[..., 0].abs() + pairs[..., 1].abs()).amax(1)
            moved = 2 * 136 * 2.0 ** -24 * abs(scale) * qh.abs().sum(1, keepdim=True) * size + 2.0 ** -18
            w = torch.softmax(scores, -1)
            out[b, heads] = w @ v
            pairs = rows(cache.v_scales).double()
            pairs = torch.where(pairs[..., :1].isnan(), 0.0, pairs)      # a NaN group counts in its own channels only
            reach = (15 * pairs[..., 0].abs() + pairs[..., 1].abs()).repeat_interleave(cache.group, 1)
            largest = (w * pairs.abs().amax((1, 2)).clamp_min(2.0 ** -60)).amax(1, keepdim=True)
            moved_w = w * moved
            bound[b, heads] = (2.0 ** -11 * (w @ reach) + moved_w @ reach + moved_w.sum(1, keepdim=True) * out[b, heads].abs()
                               + length * largest * (2.0 ** -28 + 2.0 ** -151 * v.abs().nan_to_num(0.0, 0.0).amax()))
    return out, bound + 2.0 ** -8 * (out.abs() + bound)


def case(kernels, lengths, heads, kv_heads, head_dim, group, page, seed):
    table, pages, _ = ref.scattered_table(lengths, page, 2, seed)
    cache = ref.filled_cache(kernels, pages, kv_heads, page, head_dim, group, seed)
    q = torch.randn((len(lengths), heads, head_dim), generator=torch.Generator(device=DEV).manual_seed(seed + 1), device=DEV)
    return q.to(BF16), cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)


def check(kernels, q, cache, table, lens, lengths, scale):
    out = kernels.kv4_decode(q, cache, table, lens, scale)
    want, bound = attend(q, cache, table, lengths, scale)
    assert ((out.double() - want).abs() <= bound).all()
    assert torch.equal(out, kernels.kv4_decode(q, cache, table, lens, scale))
    assert kernels.device_status() == 0
    return out


# rows that one block holds whole, rows cut into runs of several tiles, rows cut into single tiles
BATCHES = [([200] * 150, 4, 2), ([9000] * 8, 4, 2), ([300, 1200], 8, 1)]


@pytest.mark.parametrize("lengths,heads,kv_heads", BATCHES)
@pytest.mark.parametrize("place", [0, 133, -1])
@pytest.mark.parametrize("weight", ["none", "as much", "all"])
@pytest.mark.parametrize("power", [6, 12, 20, 40, 60])
def test_one_loud_value(kernels, lengths, heads, kv_heads, place, weight, power):
    """One position of each sequence holds values 2^power times as large as the others', and weighs nothing at
    all, as much less as it is louder, or nearly everything: the others keep their bits."""
    head_dim, group, page = 128, 64, 32
    q, cache, table, lens = case(kernels, lengths, heads, kv_heads, head_dim, group, page, power)
    q = q.abs()                          # so that a key of one value for all channels has the same score for all heads
    scale = head_dim ** -0.5
    height = scale * head_dim * math.sqrt(2 / math.pi)
    score = {"none": -700.0, "as much": -power * math.log(2), "all": 30.0 + power}[weight]
    for b, n in enumerate(lengths):
        at = place % n
        where = (table[b, at // page].long(), slice(None), at % page)
        cache.k_scales[where] = torch.tensor([0.0, score / height], dtype=BF16, device=DEV)
        cache.v_scales[where] *= 2.0 ** power
    check(kernels, q, cache, table, lens, lengths, scale)


@pytest.mark.parametrize("head_dim,group,heads", [(128, 128, 8), (128, 32, 8), (128, 32, 16), (64, 64, 16), (64, 32, 5)])
def test_one_loud_group(kernels, head_dim, group, heads):
    """Other widths and groups; only the last group of the position is loud, another position is NaN in the first."""
    lengths = [500, 129, 40]
    q, cache, table, lens = case(kernels, lengths, heads, 1, head_dim, group, 16, heads)
    for b in range(3):
        cache.v_scales[table[b, 0].long(), 0, 3, -1] *= 2.0 ** 45
        cache.k_scales[table[b, 0].long(), 0, 3] = torch.tensor([0.0, -500.0], dtype=BF16, device=DEV)
    q = q.abs()
    out = check(kernels, q, cache, table, lens, lengths, head_dim ** -0.5)
    if group < head_dim:
        pair = cache.v_scales[table[0, 1].long(), 0, 2, 0]
        pair[0], pair[1] = float("nan"), float("-inf")
        got = kernels.kv4_decode(q, cache, table, lens, head_dim ** -0.5)
        assert got[0, :, :group].isnan().all() and torch.equal(got[1:], out[1:])
        want, bound = attend(q, cache, table, lengths, head_dim ** -0.5)
        assert ((got.double() - want).abs() <= bound)[0, :, group:].all()


@pytest.mark.parametrize("power", [-75, -50, 70, 100, 118])
@pytest.mark.parametrize("head_dim,group", [(128, 128), (64, 32)])
def test_value_magnitudes(kernels, power, head_dim, group):
    lengths = [700, 64, 129, 3000]
    q, cache, table, lens = case(kernels, lengths, 8, 2, head_dim, group, 64, 3)
    cache.v_scales.mul_(2.0 ** power)
    assert check(kernels, q, cache, table, lens, lengths, head_dim ** -0.5).isfinite().all()


@pytest.mark.parametrize("value", [0.0, -3.0, 2.0 ** -100, 2.0 ** 40, 2.0 ** 126])
def test_one_value_everywhere(kernels, value):
    """Groups of one value have scale 0: the result is the value, as sums of weights that round by 2^-18 at most."""
    lengths = [1, 700, 5000]
    q, cache, table, lens = case(kernels, lengths, 4, 1, 128, 64, 64, 4)
    cache.v_scales[..., 0], cache.v_scales[..., 1] = 0, value
    out = kernels.kv4_decode(q, cache, table, lens, 0.1)
    assert ((out.double() - value).abs() <= 2.0 ** -8 * abs(value)).all()


@pytest.mark.parametrize("power", [-112, 112])
def test_query_and_key_magnitudes(kernels, power):
    """Queries of 2^power over keys of 2^-power."""
    lengths = [300, 20]
    q, cache, table, lens = case(kernels, lengths, 8, 2, 128, 64, 32, 5)
    cache.k_scales.mul_(2.0 ** -power)
    check(kernels, (q.float() * 2.0 ** power).to(BF16), cache, table, lens, lengths, 128 ** -0.5)
