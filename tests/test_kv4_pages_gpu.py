"""Page numbers outside the 4-bit cache: page 0 is read in their place (B200 only)."""
import pytest
import torch

import test_kv4_gpu as kv4_test

pytestmark = kv4_test.pytestmark
kernels = kv4_test.kernels


@pytest.mark.parametrize("bad", ["behind", "far behind", "negative", "most negative"])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_page_zero_is_read(kernels, bad, page):
    q, cache, table, lens, scale, out = kv4_test.run_attend(kernels, [600, 37, 300], 8, 2, 128, 128, page, seed=page)
    number = {"behind": cache.pages, "far behind": 2 ** 31 - 1, "negative": -1, "most negative": -2 ** 31}[bad]
    broken, replaced = table.clone(), table.clone()
    for b, place in ((0, 0), (0, table.shape[1] - 1), (2, (300 - 1) // page)):
        broken[b, place], replaced[b, place] = number, 0
    want = kernels.kv4_decode(q, cache, replaced, lens, scale)
    assert kernels.device_status() == 0
    got = kernels.kv4_decode(q, cache, broken, lens, scale)
    assert kernels.device_status(clear=True) & 0xffff == 0x903
    assert torch.equal(got, want) and torch.equal(got[1], out[1])
