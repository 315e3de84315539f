"""The serving operators behind offsets of 2^31 elements and 2^32 bytes (B200 only): rows at the end of large tensors
come out as in small ones."""
import pytest
import torch

import kv4_reference as ref
import test_adapters_gpu as adapters_test
import test_block_norm_gpu as norm_test

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    yield k
    torch.cuda.empty_cache()


@pytest.mark.parametrize("head_dim,group", [(128, 64), (64, 32)])
def test_cache(kernels, head_dim, group):
    kv_heads, page = 8, 64
    pages = 2 ** 32 // (kv_heads * page * head_dim // 2) + 40       # codes of more than 2^32 bytes
    cache = kernels.kv4_cache(pages, kv_heads, page, head_dim, group, DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    tokens = 150
    k, v = (torch.randn((tokens, kv_heads, head_dim), generator=gen, device=DEV).to(BF16) for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 30, 3], [pages - 2, 0, 0]], dtype=torch.int32, device=DEV)
    at = torch.arange(tokens, device=DEV)
    slots = table[0].long()[at // page] * page + at % page
    kernels.kv4_append(cache, k, v, slots)
    for x, codes, pairs in ((k, cache.k_codes, cache.k_scales), (v, cache.v_codes, cache.v_scales)):
        want_codes, want_pairs = ref.quantise(x, group)
        assert torch.equal(codes[slots // page, :, slots % page], ref.pack(want_codes))
        assert torch.equal(pairs[slots // page, :, slots % page], want_pairs)
    assert not cache.k_codes[5:50].any() and not cache.v_codes[:3].any()      # where 32 bits would have put them
    got = kernels.kv4_read(cache, slots, dtype=torch.float32)
    for x, out in zip((k, v), got):
        codes, pairs = ref.quantise(x, group)
        assert torch.equal(out, ref.values(ref.pack(codes), pairs, torch.float32))
    q = torch.randn((2, 16, head_dim), generator=gen, device=DEV).to(BF16)
    lengths = torch.tensor([tokens, 40], dtype=torch.int32, device=DEV)
    want, _, bound = ref.attend(q, cache, table, [tokens, 40], 0.1)
    assert ((kernels.kv4_decode(q, cache, table, lengths, 0.1).double() - want).abs() <= bound).all()
    assert kernels.device_status() == 0


def test_adapters(kernels):
    m, k, n, rank = 80001, 64, 28672, 16          # 2.29e9 elements of the output and of the contribution
    x, w, down, up, scales, bias = adapters_test.make(m, k, n, rank, 3, 1)
    index = (torch.arange(m, device=DEV) % 4 - 1).to(torch.int32)
    out = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias)
    rows = torch.cat([torch.arange(0, 3), torch.arange(m // 2, m // 2 + 5), torch.arange(74890, 74910), torch.arange(m - 70, m)]).to(DEV)
    adapters_test.check(out[rows], *adapters_test.expected(x[rows], w, down, up, index[rows], scales, bias))


@pytest.mark.parametrize("cols", [16384, 16380])
def test_seam(kernels, cols):
    rows = 2 ** 31 // cols + 700
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.empty((rows, cols), dtype=BF16, device=DEV).normal_(generator=gen)
    residual = torch.empty((rows, cols), dtype=BF16, device=DEV).normal_(generator=gen)
    h, y = kernels.rmsnorm_residual(x, residual, gate=x, eps=1e-6)
    some = torch.cat([torch.arange(0, 3), torch.arange(rows - 710, rows)]).to(DEV)
    norm_test.check(h[some], y[some], norm_test.formulas(x[some], residual[some], None, None, x[some], 1.0, 1e-6, False), None)
