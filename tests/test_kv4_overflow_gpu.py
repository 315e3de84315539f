"""Attention over the 4-bit cache where scores overflow (B200 only)."""
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


def attend(q, cache, table, lengths, scale, skip):
    """``kv4_reference.attend`` over the positions from ``skip`` on, a multiple of the page."""
    out, _, bound = ref.attend(q, cache, table[:, skip // cache.page:], [n - skip for n in lengths], scale)
    return out, bound


def case(kernels, lengths, heads, kv_heads, head_dim, group, page, seed):
    table, pages, _ = ref.scattered_table(lengths, page, 2, seed)
    cache = ref.filled_cache(kernels, pages, kv_heads, page, head_dim, group, seed)
    q = torch.randn((len(lengths), heads, head_dim), generator=torch.Generator(device=DEV).manual_seed(seed + 1), device=DEV)
    return q.to(BF16), cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV)


def check(kernels, q, cache, table, lens, lengths, scale, skip):
    out = kernels.kv4_decode(q, cache, table, lens, scale)
    want, bound = attend(q, cache, table, lengths, scale, skip)
    assert ((out.double() - want).abs() <= bound).all()
    assert torch.equal(out, kernels.kv4_decode(q, cache, table, lens, scale))
    assert kernels.device_status() == 0
    return out


@pytest.mark.parametrize("first", [16, 128, 400])
def test_scores_of_minus_infinity(kernels, first):
    """Scores that overflow downwards weigh nothing, also where a warp sees no others at first, or none at all."""
    lengths = [600, 401]
    q, cache, table, lens = case(kernels, lengths, 8, 1, 128, 64, 16, 6)
    q = q.abs()
    for b in range(2):
        cache.k_scales[table[b, : first // 16].long(), 0] = torch.tensor([0.0, -3e38], dtype=BF16, device=DEV)
    check(kernels, q, cache, table, lens, lengths, 128 ** -0.5, skip=first)
