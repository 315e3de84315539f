"""The fused block seam (post norm, gate, residual, next norm) against the formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


def formulas(x, residual, gain, post_gain, gate, scale, eps, post_norm):
    """h, y and, for the bound, the sum of the magnitudes that h is the difference of."""
    b = x.double()
    if post_norm:
        b = b / torch.sqrt(b.square().mean(1, keepdim=True) + eps)
        if post_gain is not None:
            b = b * post_gain.double()
    if gate is not None:
        b = b * gate.double()
    r = residual.double() * scale
    h = r + b
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
    if gain is not None:
        y = y * gain.double()
    return h, y, r.abs() + b.abs()


def check(h, y, expected, gain):
    """A lane adds 16 squares one after the other, then at most five shuffles and 32 warps follow: at
    most 53 roundings of 2^-24 of a sum of squares, halved by the square root, and six more
    (division, root, three products, the addition): 2^-19 of |residual part| + |gate part| covers h
    before its own rounding.  That error reaches y through the element and through the row's norm."""
    want_h, want_y, size = expected
    slack = 2.0 ** -19
    dh = slack * size
    rounding = torch.finfo(h.dtype).eps / 2
    assert ((h.double() - want_h).abs() <= dh + rounding * (want_h.abs() + dh)).all()
    norm = want_h.norm(dim=1, keepdim=True).clamp_min(1e-300)
    rel = dh.norm(dim=1, keepdim=True) / norm + slack
    inv = want_y.abs() / want_h.abs().clamp_min(1e-300)
    dy = dh * inv + rel * want_y.abs()
    assert ((y.double() - want_y).abs() <= dy + 2.0 ** -8 * (want_y.abs() + dy) + 1e-38).all()


def make(rows, cols, x_dtype, residual_dtype, gate_kind, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    x, residual = rand(rows, cols).to(x_dtype), (2 * rand(rows, cols)).to(residual_dtype)
    gain, post_gain = (1 + 0.25 * rand(cols)).to(BF16), (1 + 0.25 * rand(cols)).to(BF16)
    shape = {"none": None, "vector": (cols,), "column": (1, cols), "row": (rows, 1), "full": (rows, cols)}[gate_kind]
    gate = None if shape is None else (0.5 * rand(*shape)).to(BF16)
    return x, residual, gain, post_gain, gate


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 511), (5, 512), (3, 520), (9, 1000), (4, 1024), (2, 1025),
                                       (3, 2055), (2, 4096), (1, 4100), (2, 8192), (1, 8193), (2, 16384), (1, 16383),
                                       (131, 64), (257, 136)])
@pytest.mark.parametrize("x_dtype,residual_dtype", [(BF16, BF16), (BF16, FP32), (FP32, BF16), (FP32, FP32)])
def test_sizes_and_types(kernels, rows, cols, x_dtype, residual_dtype):
    x, residual, gain, post_gain, gate = make(rows, cols, x_dtype, residual_dtype, "vector", rows * 7 + cols)
    h, y = kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, gate=gate, residual_scale=0.75, eps=1e-6)
    assert h.dtype == residual_dtype and y.dtype == BF16
    check(h, y, formulas(x, residual, gain, post_gain, gate, 0.75, 1e-6, True), gain)


@pytest.mark.parametrize("gate_kind", ["none", "vector", "column", "row", "full"])
@pytest.mark.parametrize("post", ["none", "norm", "gain"])
@pytest.mark.parametrize("cols", [520, 77])
def test_gates_and_post_norms(kernels, gate_kind, post, cols):
    x, residual, gain, post_gain, gate = make(37, cols, BF16, BF16, gate_kind, 5)
    use = post_gain if post == "gain" else None
    h, y = kernels.rmsnorm_residual(x, residual, gain=None if post == "norm" else gain, post_gain=use,
                                    post_norm=post != "none", gate=gate, eps=1e-5)
    check(h, y, formulas(x, residual, None if post == "norm" else gain, use, gate, 1.0, 1e-5, post != "none"), gain)


@pytest.mark.parametrize("pitch,offset", [(640, 0), (641, 0), (640, 8), (640, 3)])
def test_strided_operands(kernels, pitch, offset):
    """Views with a row pitch, and (odd pitch or offset) rows that do not start on 16 bytes."""
    rows, cols = 19, 512
    x, residual, gain, post_gain, gate = make(rows, cols, BF16, FP32, "full", 8)

    def view(t):
        wide = torch.full((rows, pitch), 7.0, dtype=t.dtype, device=DEV)
        wide[:, offset:offset + cols] = t
        return wide, wide[:, offset:offset + cols]

    (_, xv), (_, rv), (_, gv) = view(x), view(residual), view(gate)
    wide_h, hv = view(torch.zeros_like(residual))
    wide_y, yv = view(torch.zeros_like(x))
    kernels.rmsnorm_residual(xv, rv, gain=gain, post_gain=post_gain, gate=gv, eps=1e-6, residual_out=hv, out=yv)
    check(hv, yv, formulas(x, residual, gain, post_gain, gate, 1.0, 1e-6, True), gain)
    for wide in (wide_h, wide_y):      # what lies between the rows stays
        assert (wide[:, :offset] == 7).all() and (wide[:, offset + cols:] == 7).all()


@pytest.mark.parametrize("cols", [1024, 1001])
def test_in_place(kernels, cols):
    x, residual, gain, post_gain, gate = make(65, cols, BF16, BF16, "full", 11)
    want = kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, gate=gate, eps=1e-6)
    x2, r2 = x.clone(), residual.clone()
    h, y = kernels.rmsnorm_residual(x2, r2, gain=gain, post_gain=post_gain, gate=gate, eps=1e-6, residual_out=r2, out=x2)
    assert h is r2 and y is x2 and torch.equal(h, want[0]) and torch.equal(y, want[1])


def test_special_values_stay_in_their_row(kernels):
    x, residual, gain, post_gain, gate = make(6, 264, BF16, BF16, "none", 3)
    clean = kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, eps=1e-6)
    x[1, 5], x[2, 0], residual[3, 9] = float("nan"), float("inf"), float("-inf")
    h, y = kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, eps=1e-6)
    for row in (0, 4, 5):
        assert torch.equal(h[row], clean[0][row]) and torch.equal(y[row], clean[1][row])
    assert y[1].isnan().all()
    assert h[2, 0].isnan() and y[2].isnan().all()          # inf / inf under the post norm
    assert h[3, 9] == float("-inf") and y[3, 9].isnan() and (y[3, :9] == 0).all()
    # nothing but zeros: 0 / sqrt(0 + eps) is 0, and 0 / 0 is NaN without eps
    zero = torch.zeros(2, 64, dtype=BF16, device=DEV)
    assert (kernels.rmsnorm_residual(zero, zero, eps=1e-6)[1] == 0).all()
    assert kernels.rmsnorm_residual(zero, zero, eps=0.0)[1].isnan().all()


def test_other_stream_and_graph(kernels):
    x, residual, gain, post_gain, gate = make(64, 2048, BF16, FP32, "column", 21)
    want = kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, gate=gate, eps=1e-6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, gate=gate, eps=1e-6, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    h, y = torch.empty_like(residual), torch.empty_like(x)
    with torch.cuda.graph(graph):
        kernels.rmsnorm_residual(x, residual, gain=gain, post_gain=post_gain, gate=gate, eps=1e-6, residual_out=h, out=y)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    check(h, y, formulas(x, residual, gain, post_gain, gate, 1.0, 1e-6, True), gain)


def test_refusals(kernels):
    x = torch.zeros(4, 64, dtype=BF16, device=DEV)
    for call in (lambda: kernels.rmsnorm_residual(x, x[:2]), lambda: kernels.rmsnorm_residual(x.half(), x),
                 lambda: kernels.rmsnorm_residual(x, x, gate=x[:, :8]), lambda: kernels.rmsnorm_residual(x, x, gain=x[0, :8]),
                 lambda: kernels.rmsnorm_residual(x, x, post_gain=x[0], post_norm=False),
                 lambda: kernels.rmsnorm_residual(x, x, residual_out=torch.zeros(4, 64, device=DEV)),
                 lambda: kernels.rmsnorm_residual(x.t(), x.t())):
        with pytest.raises(ValueError):
            call()
    wide = torch.zeros(1, 16385, dtype=BF16, device=DEV)
    for call in (lambda: kernels.rmsnorm_residual(wide, wide), lambda: kernels.rmsnorm_residual(x[:0], x[:0]),
                 lambda: kernels.rmsnorm_residual(x, x[:1].expand(4, 64))):
        with pytest.raises(kernels.KernelError):
            call()
