"""Operands of one row, one head or one adapter inside tensors of any pitch (B200 only): the bits of contiguous copies."""
import pytest
import torch

import kv4_reference as ref
import test_adapters_gpu as adapters_test

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


def odd(t, axis):
    """``t``, of one entry along ``axis``, with an odd stride there."""
    strides = list(t.contiguous().stride())
    strides[axis] = 2 * t.numel() + 3
    return t.contiguous().as_strided(t.shape, strides)


def test_adapters(kernels):
    x, w, down, up, scales, bias = adapters_test.make(1, 264, 136, 16, 1, 3)
    index = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias)
    out = odd(torch.empty_like(want), 0)
    got = kernels.gemm_adapters(odd(x, 0), w, odd(down, 0), odd(up, 0), index, scales=scales, bias=bias, out=out)
    assert got is out and torch.equal(got, want)


def test_seam(kernels):
    x = torch.randn(1, 264, device=DEV).to(BF16)
    want = kernels.rmsnorm_residual(x, x, gate=x, eps=1e-6)
    got = kernels.rmsnorm_residual(odd(x, 0), odd(x, 0), gate=odd(x, 0), eps=1e-6, out=odd(torch.empty_like(x), 0))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tokens,kv_heads", [(1, 2), (5, 1), (1, 1)])
def test_cache(kernels, tokens, kv_heads):
    k, v = (torch.randn(tokens, kv_heads, 128, device=DEV).to(BF16) for _ in range(2))
    slots = torch.arange(tokens, device=DEV)
    caches = [kernels.kv4_cache(2, kv_heads, 16, 128, 64, DEV) for _ in range(2)]
    axes = [axis for axis, n in enumerate((tokens, kv_heads)) if n == 1]
    kernels.kv4_append(caches[0], k, v, slots)
    for axis in axes:
        kernels.kv4_append(caches[1], odd(k, axis), odd(v, axis), slots)
        assert all(torch.equal(a, b) for a, b in zip(caches[0].tensors, caches[1].tensors))
        want = kernels.kv4_read(caches[0], slots)
        outs = [odd(torch.empty_like(k), axis) for _ in range(2)]
        kernels.kv4_read(caches[0], slots, k_out=outs[0], v_out=outs[1])
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("batch,heads", [(1, 4), (3, 1), (1, 1)])
def test_decode(kernels, batch, heads):
    lengths = [70] * batch
    table, pages, _ = ref.scattered_table(lengths, 16, 1, 1)
    cache = ref.filled_cache(kernels, pages, 1, 16, 128, 64, 1)
    q = torch.randn(batch, heads, 128, device=DEV).to(BF16)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = kernels.kv4_decode(q, cache, table, lens, 0.1)
    for axis in [axis for axis, n in enumerate((batch, heads)) if n == 1]:
        assert torch.equal(kernels.kv4_decode(odd(q, axis), cache, table, lens, 0.1), want)
