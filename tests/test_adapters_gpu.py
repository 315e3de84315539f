"""GEMM with low-rank adapters per row against 64 bits (B200 only)."""
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


def make(m, k, n, rank, count, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    x, w = rand(m, k).to(BF16), (rand(k, n) * k ** -0.5).to(BF16)
    down, up = (rand(count, k, rank) * k ** -0.5).to(BF16), (rand(count, rank, n) * rank ** -0.5).to(BF16)
    return x, w, down, up, 0.5 + torch.rand(count, generator=gen, device=DEV), rand(n).to(BF16)


def expected(x, w, down, up, index, scales, bias):
    """The result in 64 bits and the bound of the error before the last rounding.

    scale * (x down) is rounded to BF16 (2^-8 of each |t|, which reaches the result through |up|), and so
    is the contribution with the bias (2^-8 of it).  A sum of k products in FP32 is off by at most
    k 2^-24 of the sum of their magnitudes, the one of `rank` products by rank 2^-24."""
    x64, w64 = x.double(), w.double()
    out = x64 @ w64
    m, k = x.shape
    slack = k * 2.0 ** -24 * (x64.abs() @ w64.abs())
    delta, bound = torch.zeros_like(out), torch.zeros_like(out)
    for z in range(down.shape[0]):
        rows = (index == z).nonzero().flatten()
        if len(rows) == 0:
            continue
        s = 1.0 if scales is None else scales[z].double()
        d, u = down[z].double(), up[z].double()
        t = s * (x64[rows] @ d)
        dt = 2.0 ** -8 * t.abs() + 2 * k * 2.0 ** -24 * s * (x64[rows].abs() @ d.abs())
        delta[rows] = t @ u
        bound[rows] = dt @ u.abs() + down.shape[2] * 2.0 ** -24 * ((t.abs() + dt) @ u.abs())
    if bias is not None:
        delta = delta + bias.double()
    bound = bound + 2.0 ** -8 * (delta.abs() + bound)
    return out + delta, bound + slack + 2.0 ** -23 * (out.abs() + delta.abs())


def check(got, want, bound):
    rounding = torch.finfo(got.dtype).eps / 2
    assert ((got.double() - want).abs() <= bound + rounding * (want.abs() + bound)).all()


def indexes(kind, m, count, seed=0):
    gen = torch.Generator().manual_seed(seed)
    if kind == "mixed":
        index = torch.randint(-1, count, (m,), generator=gen)
    elif kind == "sorted":
        index = torch.randint(-1, count, (m,), generator=gen).sort().values
    elif kind == "none":
        index = torch.full((m,), -1)
    elif kind == "one":
        index = torch.full((m,), count - 1)
    else:
        index = torch.arange(m) % count
    return index.to(torch.int32).to(DEV)


@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (1, 512, 128), (7, 136, 264), (16, 1024, 384), (17, 1032, 1000), (33, 2048, 256),
                                   (64, 264, 2056), (65, 520, 136), (130, 256, 640)])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 64, 72, 128])
def test_sizes_and_ranks(kernels, m, k, n, rank):
    x, w, down, up, scales, bias = make(m, k, n, rank, 5, m + k + n + rank)
    index = indexes("mixed", m, 5, rank)
    check(kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias),
          *expected(x, w, down, up, index, scales, bias))


@pytest.mark.parametrize("kind", ["mixed", "sorted", "none", "one", "cycle"])
@pytest.mark.parametrize("count", [1, 3, 40, 200])
@pytest.mark.parametrize("m", [16, 100])
def test_assignments(kernels, kind, count, m):
    x, w, down, up, scales, _ = make(m, 384, 320, 16, count, count)
    index = indexes(kind, m, count)
    check(kernels.gemm_adapters(x, w, down, up, index, scales=scales), *expected(x, w, down, up, index, scales, None))


@pytest.mark.parametrize("most", [15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64])
@pytest.mark.parametrize("rank,n", [(16, 328), (64, 264), (128, 520)])
def test_shares_of_a_tile(kernels, most, rank, n):
    """Rows of one adapter scattered over a tile of 64 rows in every number of sixteens, others and none between;
    a bias reaches the rows without an adapter too; few tiles of rows and many."""
    for m in (64, 333):
        x, w, down, up, scales, bias = make(m, 136, n, rank, 4, most)
        index = indexes("mixed", m, 3, most)
        for row0 in range(0, m, 64):
            places = row0 + torch.randperm(64, generator=torch.Generator().manual_seed(row0 + most))[:most]
            index[places[places < m].to(DEV)] = 3
        check(kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias),
              *expected(x, w, down, up, index, scales, bias))


@pytest.mark.parametrize("m", [4735, 4736, 5000])
@pytest.mark.parametrize("kind", ["mixed", "sorted"])
def test_prompts(kernels, m, kind):
    """Both row tiles of the first kernel; many tiles, the last one partly filled."""
    for rank in (16, 128):
        x, w, down, up, scales, bias = make(m, 512, 264, rank, 9, m)
        index = indexes(kind, m, 9)
        check(kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias),
              *expected(x, w, down, up, index, scales, bias))


def test_long_inner_axis(kernels):
    x, w, down, up, scales, _ = make(5, 28672, 128, 64, 2, 3)
    index = indexes("cycle", 5, 2)
    check(kernels.gemm_adapters(x, w, down, up, index), *expected(x, w, down, up, index, None, None))


@pytest.mark.parametrize("activation", ["relu", "silu"])
def test_activation_and_fp32(kernels, activation):
    x, w, down, up, scales, bias = make(33, 256, 136, 16, 4, 1)
    index = indexes("mixed", 33, 4)
    act = kernels.ACT_RELU if activation == "relu" else kernels.ACT_SILU
    want, bound = expected(x, w, down, up, index, scales, bias)
    got = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias, activation=act, out_dtype=torch.float32)
    full = want.relu() if activation == "relu" else torch.nn.functional.silu(want)
    # the slope of either is below 1.1; the epilogue's sigmoid is good to 2^-20
    check(got, full, 1.1 * bound + 2.0 ** -20 * want.abs())


def test_views(kernels):
    """Operands and output inside wider tensors."""
    m, k, n, rank, count = 21, 264, 56, 16, 3
    x, w, down, up, scales, bias = make(m, k, n, rank, count, 2)
    wide = lambda t, extra: torch.nn.functional.pad(t, (0, extra), value=float("nan"))
    xv, wv, dv = wide(x, 24)[:, :k], wide(w, 8)[:, :n], wide(down, 8)[..., :rank]
    uv = wide(up, 16)[..., :n]
    out = torch.full((m, 72), 5.0, dtype=BF16, device=DEV)
    index = indexes("mixed", m, count)
    kernels.gemm_adapters(xv, wv, dv, uv, index, scales=scales, bias=bias, out=out[:, :n])
    check(out[:, :n], *expected(x, w, down, up, index, scales, bias))
    assert (out[:, n:] == 5).all()


def test_bad_adapters_stay_with_their_rows(kernels):
    m, count = 50, 4
    x, w, down, up, scales, _ = make(m, 256, 200, 16, count, 4)
    index = indexes("cycle", m, count)
    clean = kernels.gemm_adapters(x, w, down, up, index, scales=scales)
    down[1, 3, 5], up[2, 7, 9], scales[3] = float("nan"), float("inf"), float("inf")
    got = kernels.gemm_adapters(x, w, down, up, index, scales=scales)
    assert torch.equal(got[index == 0], clean[index == 0])
    assert got[index == 1].isnan().all()
    others = torch.ones(200, dtype=torch.bool, device=DEV)
    others[9] = False
    assert torch.equal(got[index == 2][:, others], clean[index == 2][:, others])
    assert not got[index == 2][:, 9].isfinite().any()
    # adapters that no row names are not read
    down[1], up[2] = float("nan"), float("nan")
    index = torch.zeros_like(index)
    assert kernels.gemm_adapters(x, w, down, up, index, scales=scales).isfinite().all()


def test_index_outside(kernels):
    x, w, down, up, scales, _ = make(20, 64, 64, 8, 2, 5)
    index = indexes("cycle", 20, 2)
    bad = index.clone()
    bad[3], bad[7] = 2, 2 ** 31 - 1
    got = kernels.gemm_adapters(x, w, down, up, bad, scales=scales)
    assert kernels.device_status(clear=True) & 0xffff == 0xA01
    bad[3] = bad[7] = -1
    assert torch.equal(got, kernels.gemm_adapters(x, w, down, up, bad, scales=scales))
    assert kernels.device_status() == 0


def test_stream_graph_and_workspace(kernels):
    m = 40
    x, w, down, up, scales, bias = make(m, 512, 384, 32, 6, 6)
    index = indexes("mixed", m, 6)
    want = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias)
    room = torch.full((kernels.gemm_adapters_workspace_bytes(m, 384, 32),), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias, workspace=room), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
    with torch.cuda.graph(graph):
        for _ in range(3):
            kernels.gemm_adapters(x, w, down, up, index, scales=scales, bias=bias, out=out)
    x.neg_()
    index.copy_(indexes("cycle", m, 6))
    graph.replay()
    torch.cuda.synchronize()
    check(out, *expected(x, w, down, up, index, scales, bias))


def test_refusals(kernels):
    x, w, down, up, scales, bias = make(4, 64, 64, 16, 2, 7)
    index = indexes("cycle", 4, 2)
    for call in (lambda: kernels.gemm_adapters(x, w[:32], down, up, index),
                 lambda: kernels.gemm_adapters(x, w, down[:1], up, index),
                 lambda: kernels.gemm_adapters(x, w, down[:, :32], up, index),
                 lambda: kernels.gemm_adapters(x, w, down, up[:, :8], index),
                 lambda: kernels.gemm_adapters(x, w, down, up, index.long()),
                 lambda: kernels.gemm_adapters(x, w, down, up, index[:2]),
                 lambda: kernels.gemm_adapters(x, w, down, up, index.cpu()),
                 lambda: kernels.gemm_adapters(x, w, down, up, index, scales=scales.double()),
                 lambda: kernels.gemm_adapters(x, w, down, up, index, bias=bias[:8]),
                 lambda: kernels.gemm_adapters(x, w, down, up, index, out=torch.empty(4, 64, dtype=torch.half, device=DEV)),
                 lambda: kernels.gemm_adapters(x, w, down.half(), up, index)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: kernels.gemm_adapters(x, w, down[..., :12], up[:, :12], index),
                 lambda: kernels.gemm_adapters(x[:, :60], w[:60], down[:, :60], up, index),
                 lambda: kernels.gemm_adapters(x, w[:, :60], down, up[..., :60], index),
                 lambda: kernels.gemm_adapters(x[:0], w, down, up, index[:0]),
                 lambda: kernels.gemm_adapters(x, w, down, up, index, activation=kernels.ACT_SILU_GATE),
                 lambda: kernels.gemm_adapters(x, w, down, up, index, workspace=index)):
        with pytest.raises(kernels.KernelError):
            call()
