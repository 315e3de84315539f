"""GEMMs with a matrix side operand in every form of the kernel, also where the output takes its place (B200 only)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


def make(m, k, n, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    return rand(m, k).to(BF16), (rand(k, n) * k ** -0.5).to(BF16), (4 * rand(m, n)).to(BF16)


def check(got, a, b, side, relu):
    """k products and the side operand are added in FP32, each addition off by 2^-24 of the sum of magnitudes;
    one rounding at the end."""
    want = a.double() @ b.double() + side.double()
    slack = (a.shape[1] + 2) * 2.0 ** -24 * (a.double().abs() @ b.double().abs() + side.double().abs())
    if relu:
        want = want.relu()
    rounding = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs() <= slack + rounding * (want.abs() + slack)).all()


# CTA pairs: one unit each and not all, an odd last row tile, two and seven units each; wide, 128- and 64-column tiles;
# one row tile; the split form
SIZES = [(2048, 136, 2560), (2100, 64, 2312), (1920, 264, 5000), (4224, 64, 8200), (300, 128, 33000), (500, 520, 1000),
         (130, 64, 200), (100, 128, 30000), (64, 4096, 512), (17, 1024, 264)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("pairs", ["0", "1"])
def test_forms(kernels, monkeypatch, m, k, n, pairs):
    monkeypatch.setenv("TRINITY_SM100_GEMM_PAIRS", pairs)
    a, b, side = make(m, k, n, m + n)
    check(kernels.gemm(a, b, bias=side), a, b, side, False)
    check(kernels.gemm(a, b, bias=side, activation=kernels.ACT_RELU, out_dtype=torch.float32), a, b, side, True)
    wide = torch.full((m, n + 24), 9.0, dtype=BF16, device=DEV)      # operand and output inside wider rows
    wide[:, 8:n + 8] = side
    out = torch.full((m, n + 40), 7.0, dtype=BF16, device=DEV)
    kernels.gemm(a, b, bias=wide[:, 8:n + 8], out=out[:, 16:n + 16])
    check(out[:, 16:n + 16], a, b, side, False)
    assert (out[:, :16] == 7).all() and (out[:, n + 16:] == 7).all()


@pytest.mark.parametrize("m,k,n", SIZES)
def test_output_in_the_place_of_the_operand(kernels, m, k, n):
    a, b, side = make(m, k, n, m)
    want = kernels.gemm(a, b, bias=side)
    stream = side.clone()
    for _ in range(3):
        stream.copy_(side)
        assert kernels.gemm(a, b, bias=stream, out=stream) is stream
        assert torch.equal(stream, want)
