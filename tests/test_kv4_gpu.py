"""The 4-bit cache: its format bit by bit, attention over it against 64 bits (B200 only)."""
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


def same(a, b):
    """Equal bit patterns, NaN for NaN."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all()) if a.is_floating_point() else torch.equal(a, b)


def rows(tokens, kv_heads, head_dim, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((tokens, kv_heads, head_dim), generator=gen, device=DEV) * 3).to(BF16)


def check_cache(kernels, cache, k, v, slots, group):
    page, place = slots // cache.page, slots % cache.page
    for x, codes, scales, out in ((k, cache.k_codes, cache.k_scales, 0), (v, cache.v_codes, cache.v_scales, 1)):
        want_codes, want_pairs = ref.quantise(x, group)
        assert torch.equal(codes[page, :, place], ref.pack(want_codes))
        assert same(scales[page, :, place][..., 0], want_pairs[..., 0])
        want = ref.values(ref.pack(want_codes), want_pairs, torch.float32)
        assert same(kernels.kv4_read(cache, slots, dtype=torch.float32)[out], want)
        assert same(kernels.kv4_read(cache, slots)[out], want.to(BF16))


@pytest.mark.parametrize("head_dim,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("tokens,kv_heads,page", [(1, 1, 16), (3, 2, 48), (33, 3, 64), (257, 8, 128)])
def test_append_and_read(kernels, head_dim, group, tokens, kv_heads, page):
    pages = -(-tokens // page) + 2
    cache = kernels.kv4_cache(pages, kv_heads, page, head_dim, group, DEV)
    slots = torch.randperm(pages * page, device=DEV)[:tokens]
    slots[-1] = pages * page - 1 if not (slots == pages * page - 1).any() else slots[-1]
    k, v = rows(tokens, kv_heads, head_dim, 1), rows(tokens, kv_heads, head_dim, 2)
    kernels.kv4_append(cache, k, v, slots)
    check_cache(kernels, cache, k, v, slots, group)
    # nothing else was written
    untouched = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    untouched[slots] = False
    for t in cache.tensors:
        assert (t.transpose(1, 2).flatten(0, 1)[untouched] == 0).all()


@pytest.mark.parametrize("pitch,offset", [(24, 8), (17, 1)])
def test_append_of_views(kernels, pitch, offset):
    """Rows inside a wider projection; with an odd pitch they do not start on 16 bytes."""
    wide = rows(40, 1, 2 * 128 * 4 + pitch, 5)[:, 0]
    k = wide[:, offset:offset + 512].unflatten(1, (4, 128))
    v = wide[:, offset + 512:offset + 1024].unflatten(1, (4, 128))
    cache = kernels.kv4_cache(4, 4, 16, 128, 64, DEV)
    slots = torch.arange(3, 43, device=DEV)
    kernels.kv4_append(cache, k, v, slots)
    check_cache(kernels, cache, k, v, slots, 64)


@pytest.mark.parametrize("pad", [0, 8, 1])
@pytest.mark.parametrize("head_dim,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
def test_many_rows(kernels, head_dim, group, pad):
    """Enough rows to fill the GPU, which start on 32, 16 or 2 bytes; some of them are padding, some lie outside."""
    kv_heads, page, tokens = 3, 48, 331000 // (3 * head_dim // 8)
    wide = rows(tokens, 2 * kv_heads, head_dim + pad, 21)
    wide[7, :, 5] = float("nan")
    wide[9] *= 2.0 ** -125                         # scales that are divided by, and subnormal values
    wide[11, :, 40] = float("inf")
    k, v = wide[:, :kv_heads, pad:], wide[:, kv_heads:, pad:]
    pages = tokens // page + 2
    cache = kernels.kv4_cache(pages, kv_heads, page, head_dim, group, DEV)
    slots = torch.randperm(pages * page, device=DEV)[:tokens]
    left_out = torch.arange(tokens, device=DEV) % 7 == 3
    slots[left_out] = -1
    kernels.kv4_append(cache, k, v, slots)
    check_cache(kernels, cache, k[~left_out], v[~left_out], slots[~left_out], group)
    written = torch.zeros(pages * page, dtype=torch.bool, device=DEV)
    written[slots[~left_out]] = True
    for t in cache.tensors:
        assert (t.transpose(1, 2).flatten(0, 1)[~written] == 0).all()
    room = 8 if pad else 0                         # outputs inside wider rows that start on 16 bytes
    for dtype in (BF16, torch.float32):
        outs = [torch.full((tokens, kv_heads, head_dim + room), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
        kernels.kv4_read(cache, slots, dtype=dtype, k_out=outs[0][..., room:], v_out=outs[1][..., room:])
        whole = kernels.kv4_read(cache, slots.abs(), dtype=dtype)
        for out, other in zip(outs, whole):
            assert (out[left_out][..., room:] == 0).all() and (out[..., :room] == 7).all()
            assert same(out[~left_out][..., room:], other[~left_out])
    assert kernels.device_status() == 0
    slots[-1], slots[100] = pages * page, 2 ** 40
    before = [t.clone() for t in cache.tensors]
    kernels.kv4_append(cache, v, k, torch.where(slots < pages * page, -1, slots))
    torch.cuda.synchronize()
    assert kernels.device_status(clear=True) & 0xffff == 0x901
    assert all(same(a, b) for a, b in zip(before, cache.tensors))


def test_padding_and_slots_outside(kernels):
    k, v = rows(6, 2, 64, 7), rows(6, 2, 64, 8)
    cache = kernels.kv4_cache(2, 2, 16, 64, 32, DEV)
    slots = torch.tensor([5, -1, 31, -7, 0, -1], device=DEV)
    kernels.kv4_append(cache, k, v, slots)
    kept = torch.tensor([0, 2, 4], device=DEV)
    check_cache(kernels, cache, k[kept], v[kept], slots[kept], 32)
    back = kernels.kv4_read(cache, slots)
    assert (back[0][1] == 0).all() and (back[1][5] == 0).all()
    assert kernels.device_status() == 0
    before = [t.clone() for t in cache.tensors]
    kernels.kv4_append(cache, k, v, torch.tensor([32, -1, 1 << 40, -1, -1, -1], device=DEV))
    assert kernels.device_status(clear=True) & 0xffff == 0x901
    assert all(torch.equal(a, b) for a, b in zip(before, cache.tensors))
    back = kernels.kv4_read(cache, torch.tensor([32, 5], device=DEV))
    assert kernels.device_status(clear=True) & 0xffff == 0x902 and (back[0][0] == 0).all() and (back[0][1] != 0).any()


def test_special_values(kernels):
    k = rows(8, 1, 128, 9)
    k[0] = 1.25                                    # one value only
    k[1, 0, 3] = float("inf")
    k[2, 0, 70] = float("nan")
    k[3, 0, 0], k[3, 0, 1] = 3e38, -3e38           # the spread overflows
    k[4] = 0
    k[5] *= 2.0 ** -130                            # subnormal scale
    k[6, 0, :64] = 0
    k[7, 0, 5] = -0.0
    v = rows(8, 1, 128, 10)
    cache = kernels.kv4_cache(1, 1, 16, 128, 64, DEV)
    slots = torch.arange(8, device=DEV)
    kernels.kv4_append(cache, k, v, slots)
    check_cache(kernels, cache, k, v, slots, 64)
    back = kernels.kv4_read(cache, slots)[0]
    assert (back[0] == 1.25).all() and (back[4] == 0).all()
    assert back[1, 0, :64].isnan().all() and not back[1, 0, 64:].isnan().any()
    assert back[2, 0, 64:].isnan().all() and not back[2, 0, :64].isnan().any()
    assert back[3, 0, :64].isnan().all()


def run_attend(kernels, batch_lengths, heads, kv_heads, head_dim, group, page, seed=0, scale=None, spread=1.0):
    table, pages, _ = ref.scattered_table(batch_lengths, page, 2, seed)
    cache = ref.filled_cache(kernels, pages, kv_heads, page, head_dim, group, seed, spread=spread)
    gen = torch.Generator(device=DEV).manual_seed(seed + 1)
    q = torch.randn((len(batch_lengths), heads, head_dim), generator=gen, device=DEV).to(BF16)
    lengths = torch.tensor(batch_lengths, dtype=torch.int32, device=DEV)
    scale = head_dim ** -0.5 if scale is None else scale
    lse = torch.empty((len(batch_lengths), heads), device=DEV)
    out = kernels.kv4_decode(q, cache, table, lengths, scale, lse=lse)
    want, want_lse, bound = ref.attend(q, cache, table, batch_lengths, scale)
    assert ((out.double() - want).abs() <= bound).all()
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isneginf(lse), empty)
    # the log of the sum moves by at most the scores' error, and is rounded to FP32
    assert ((lse.double() - want_lse).abs()[~empty] <= 2.0 ** -9 + 2.0 ** -20 * want_lse[~empty].abs()).all()
    assert torch.equal(out, kernels.kv4_decode(q, cache, table, lengths, scale))   # the same bits again
    assert kernels.device_status() == 0
    return q, cache, table, lengths, scale, out


@pytest.mark.parametrize("head_dim,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 1), (14, 2), (48, 3), (40, 2), (33, 1)])
def test_head_layouts(kernels, head_dim, group, heads, kv_heads):
    run_attend(kernels, [77, 1, 300], heads, kv_heads, head_dim, group, 32, seed=heads)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 112, 128, 256])
@pytest.mark.parametrize("head_dim,group", [(128, 64), (64, 32)])
def test_pages_and_lengths(kernels, page, head_dim, group):
    run_attend(kernels, [0, 1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000, 0, 0], 16, 2, head_dim, group, page, seed=page)


@pytest.mark.parametrize("batch_lengths", [[0], [1], [0, 0, 0], [4097], [20000], [1] * 700, [129] * 37, [5000, 1, 0, 3],
                                           [0] * 400 + [33] + [0] * 300 + [2000]])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (32, 8), (32, 2)])
def test_batches(kernels, batch_lengths, heads, kv_heads):
    """Empty, single, long and many sequences: runs that cut rows everywhere and runs that are empty."""
    run_attend(kernels, batch_lengths, heads, kv_heads, 64, 64, 64, seed=3)


def test_long_averages(kernels):
    """Weights so even that the values average to almost nothing: what is left must not drown in sums that
    cancel.  The output's rounding is at most half a step of 2^-7, uniformly spread: 2^-8 / sqrt(3) =
    0.0023 in the mean square.  The rounding of weight times scale, 2^-11 / sqrt(3), reaches a
    position's code minus 8, at most 8 steps of about 0.35 where its value is about 1: 0.0008.  Together 0.0024."""
    table, pages, _ = ref.scattered_table([200000], 128, 1, 8)
    cache = ref.filled_cache(kernels, pages, 1, 128, 128, 64, 8)
    q = torch.randn((1, 8, 128), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(BF16)
    lengths = torch.tensor([200000], dtype=torch.int32, device=DEV)
    out = kernels.kv4_decode(q, cache, table, lengths, 0.01).double()
    want, _, _ = ref.attend(q, cache, table, [200000], 0.01)
    assert want.abs().mean() < 0.02 and (out - want).norm() <= 0.0024 * want.norm()


@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.1, 1.0), (3.0, 4.0), (0.088, 2.0 ** -60), (2.0 ** -40, 2.0 ** 40)])
def test_scales(kernels, scale, spread):
    """Equal weights, a negative scale, weights concentrated on few positions, tiny and large caches."""
    run_attend(kernels, [700, 64, 129], 16, 2, 128, 32, 64, seed=5, scale=scale, spread=spread)


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -30, 2.0 ** 30, 2.0 ** 118])
def test_query_magnitudes(kernels, size):
    """The query enters as FP16 times a power of two for each head: one head stays at size 1."""
    table, pages, _ = ref.scattered_table([150], 32, 1, 4)
    cache = ref.filled_cache(kernels, pages, 1, 32, 128, 64, 4, spread=1.0 / 64)
    q = torch.randn((1, 4, 128), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    q[:, 1:3] *= size
    q = q.to(BF16)
    scale = min(1.0, 1.0 / size)
    lengths = torch.tensor([150], dtype=torch.int32, device=DEV)
    out = kernels.kv4_decode(q, cache, table, lengths, scale)
    want, _, bound = ref.attend(q, cache, table, [150], scale)
    assert ((out.double() - want).abs() <= bound).all()


def test_values_behind_the_sequence_do_not_matter(kernels):
    """NaN scales and full codes in unused places of the last page, in other pages, and NaN entries."""
    lengths = [130, 17, 64, 0]
    q, cache, table, lens, scale, out = run_attend(kernels, lengths, 16, 2, 128, 64, 64, seed=9)
    live = torch.zeros((cache.pages, cache.page), dtype=torch.bool, device=DEV)
    for b, n in enumerate(lengths):
        for i in range(-(-n // 64)):
            live[table[b, i].long(), : min(64, n - 64 * i)] = True
    for t in cache.tensors:
        t.transpose(1, 2)[~live] = 255 if t.dtype == torch.uint8 else float("nan")
    assert torch.equal(kernels.kv4_decode(q, cache, table, lens, scale), out)


def test_nan_stays_with_its_sequence_and_head(kernels):
    q, cache, table, lens, scale, out = run_attend(kernels, [100, 200, 50], 16, 2, 128, 64, 64, seed=11)
    q2 = q.clone()
    q2[0, 3, 7] = float("nan")
    q2[2, 9, 0] = float("inf")
    got = kernels.kv4_decode(q2, cache, table, lens, scale)
    mask = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
    mask[0, 3] = mask[2, 9] = False
    assert torch.equal(got[mask], out[mask]) and got[0, 3].isnan().all() and got[2, 9].isnan().all()
    cache.k_scales[table[1, 1].long(), 1, 5, 0, 0] = float("nan")      # position 69 of sequence 1, cached head 1
    cache.v_scales[table[0, 0].long(), 0, 9, 1, 0] = float("nan")      # second group of a value of sequence 0
    got = kernels.kv4_decode(q, cache, table, lens, scale)
    assert got[1, 8:].isnan().all() and got[0, :8, 64:].isnan().all()
    assert torch.equal(got[1, :8], out[1, :8]) and torch.equal(got[2], out[2]) and torch.equal(got[0, 8:], out[0, 8:])
    assert torch.equal(got[0, :8, :64], out[0, :8, :64])


def test_page_outside_the_cache(kernels):
    q, cache, table, lens, scale, out = run_attend(kernels, [100, 200], 8, 2, 128, 128, 64, seed=12)
    bad = table.clone()
    bad[0, 1] = cache.pages
    got = kernels.kv4_decode(q, cache, bad, lens, scale)
    assert kernels.device_status(clear=True) & 0xffff == 0x903
    assert torch.equal(got[1], out[1])
    bad[0, 1] = -1
    kernels.kv4_decode(q, cache, bad, lens, scale)
    assert kernels.device_status(clear=True) & 0xffff == 0x903


def test_lengths_outside_the_table(kernels):
    q, cache, table, lens, scale, out = run_attend(kernels, [128, 128], 8, 2, 64, 32, 64, seed=13)
    many = torch.tensor([10 ** 6, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    assert torch.equal(kernels.kv4_decode(q, cache, table, many, scale), out)
    none = torch.tensor([-1, -2 ** 31], dtype=torch.int32, device=DEV)
    assert (kernels.kv4_decode(q, cache, table, none, scale) == 0).all()


def test_views_workspace_stream_and_graph(kernels):
    lengths = [900, 3, 129]
    q, cache, table, lens, scale, out = run_attend(kernels, lengths, 16, 4, 128, 64, 64, seed=14)
    fused = torch.zeros((3, 16 * 128 + 64), dtype=BF16, device=DEV)
    fused[:, 64:] = q.flatten(1)
    view = fused[:, 64:].unflatten(1, (16, 128))
    wide = torch.zeros((3, table.shape[1] + 5), dtype=torch.int32, device=DEV)
    wide[:, : table.shape[1]] = table
    room = torch.full((kernels.kv4_decode_workspace_bytes(16, 4, 128),), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(kernels.kv4_decode(view, cache, wide[:, : table.shape[1]], lens, scale, workspace=room), out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kernels.kv4_decode(q, cache, table, lens, scale, stream=side)
    side.synchronize()
    assert torch.equal(got, out)
    # a captured step follows the lengths and the cache that it finds when it is replayed
    graph = torch.cuda.CUDAGraph()
    static = torch.empty_like(out)
    k, v = rows(3, 4, 128, 31), rows(3, 4, 128, 32)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)
    lens2 = torch.zeros_like(lens)
    with torch.cuda.graph(graph):
        kernels.kv4_append(cache, k, v, slots)
        kernels.kv4_decode(q, cache, table, lens2, scale, out=static)
    for step in range(3):
        now = [n - 2 + step for n in lengths]
        place = [n - 1 for n in now]
        slots.copy_(torch.tensor([int(table[b, p // 64]) * 64 + p % 64 for b, p in enumerate(place)]))
        lens2.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        want, _, bound = ref.attend(q, cache, table, now, scale)
        assert ((static.double() - want).abs() <= bound).all()


def test_two_calls_at_once(kernels):
    """Two streams, each call with its own workspace."""
    a = run_attend(kernels, [3000] * 4, 32, 8, 128, 64, 64, seed=15)
    b = run_attend(kernels, [777] * 9, 32, 8, 128, 64, 64, seed=16)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for stream, case in zip(streams, (a, b)):
            got.append((kernels.kv4_decode(*case[:5], stream=stream), case[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


def test_refusals(kernels):
    cache = kernels.kv4_cache(4, 2, 32, 128, 64, DEV)
    q = torch.zeros(2, 8, 128, dtype=BF16, device=DEV)
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    k = torch.zeros(3, 2, 128, dtype=BF16, device=DEV)
    slots = torch.arange(3, device=DEV)
    for call in (lambda: kernels.kv4_decode(q[..., :64], cache, table, lens, 1.0),
                 lambda: kernels.kv4_decode(q, cache, table.long(), lens, 1.0),
                 lambda: kernels.kv4_decode(q, cache, table[:1], lens, 1.0),
                 lambda: kernels.kv4_decode(q, cache, table, lens.cpu(), 1.0),
                 lambda: kernels.kv4_decode(q.half(), cache, table, lens, 1.0),
                 lambda: kernels.kv4_decode(q, cache, table, lens, 1.0, out=q.float()),
                 lambda: kernels.kv4_append(cache, k[:, :1], k[:, :1], slots),
                 lambda: kernels.kv4_append(cache, k, k, slots.int()),
                 lambda: kernels.kv4_append(cache, k, k, slots[:2]),
                 lambda: kernels.kv4_read(cache, slots, dtype=torch.float16),
                 lambda: kernels.kv4_read(cache, slots, k_out=torch.empty_like(k)),
                 lambda: kernels.Kv4Cache(cache.k_codes, cache.k_scales, cache.v_codes[:2], cache.v_scales),
                 lambda: kernels.kv4_cache(4, 2, 32, 128, 48, DEV)):
        with pytest.raises(ValueError):
            call()
    odd = kernels.kv4_cache(2, 1, 24, 128, 64, DEV)
    wide = kernels.kv4_cache(2, 1, 16, 96, 32, DEV)
    for call in (lambda: kernels.kv4_append(odd, k[:, :1], k[:, :1], slots),
                 lambda: kernels.kv4_append(wide, k[:, :1, :96], k[:, :1, :96], slots),
                 lambda: kernels.kv4_append(cache, k[:0], k[:0], slots[:0]),
                 lambda: kernels.kv4_decode(q[:, :7], cache, table, lens, 1.0),
                 lambda: kernels.kv4_decode(q, cache, table, lens, 1.0, workspace=slots[:2])):
        with pytest.raises(kernels.KernelError):
            call()
