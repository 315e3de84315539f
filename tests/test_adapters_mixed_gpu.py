"""Many adapters in any order on the tiles of 64 rows that long batches take (B200 only)."""
import pytest
import torch

import test_adapters_gpu as adapters_test

pytestmark = adapters_test.pytestmark
kernels = adapters_test.kernels


@pytest.mark.parametrize("m", [4736, 4801])
@pytest.mark.parametrize("count", [2, 5, 64, 200])
@pytest.mark.parametrize("rank", [8, 64, 128])
def test_long_mixed_batches(kernels, m, count, rank):
    """The contribution is rounded by 2^-8 of itself, whatever the bias, which is added in FP32: the bound without a
    bias and the roundings of two FP32 additions.  (2^-8 of contribution plus bias would be too little
    where the two cancel.)"""
    x, w, down, up, scales, bias = adapters_test.make(m, 264, 136, rank, count, count)
    for kind in ("mixed", "cycle", "none"):
        index = adapters_test.indexes(kind, m, count)
        got = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias, out_dtype=torch.bfloat16)
        want, bound = adapters_test.expected(x, w, down, up, index, scales, None)
        full = want + bias.double()
        adapters_test.check(got, full, bound + 2.0 ** -23 * (full.abs() + bias.double().abs()))
