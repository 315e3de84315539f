"""The bias of a GEMM with adapters is added in FP32, like that of a plain GEMM (B200 only)."""
import pytest
import torch

import test_adapters_gpu as adapters_test

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


# the split form with its three numbers of rows, one tile of rows, single CTAs, CTA pairs
@pytest.mark.parametrize("m,k,n", [(5, 1024, 264), (30, 2048, 520), (61, 1024, 264), (100, 128, 328), (300, 136, 264),
                                   (300, 64, 20000)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_large_bias(kernels, m, k, n, out_dtype):
    """Against the bound without a bias: what the bias adds to it is the rounding of FP32 sums, and a
    difference of the FP32 result from the bias keeps the adapters' part."""
    x, w, down, up, scales, bias = adapters_test.make(m, k, n, 16, 3, m)
    bias = (bias * 512).to(torch.bfloat16)
    index = adapters_test.indexes("mixed", m, 3)
    got = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias, out_dtype=out_dtype)
    want, bound = adapters_test.expected(x, w, down, up, index, scales, None)
    full = want + bias.double()
    adapters_test.check(got, full, bound + 2.0 ** -23 * (full.abs() + bias.double().abs()))
