"""The 4-bit cache and its attention in plain torch: the format bit by bit, the attention in 64 bits."""
import torch


def quantise(x, group):
    """codes uint8 [..., D] and pairs BF16 [..., D / group, 2] of BF16 values [..., D]."""
    parts = x.float().unflatten(-1, (-1, group))
    low, high = parts.amin(-1, keepdim=True), parts.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(torch.bfloat16)
    bad = ~torch.isfinite(parts).all(-1, keepdim=True) | ~torch.isfinite(high - low)
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    ratio = (parts - low) / scale.float()
    codes = torch.where(scale.float() > 0, torch.round(ratio).clamp(0, 15), torch.zeros_like(parts))
    return codes.to(torch.uint8).flatten(-2), torch.cat([scale, low.to(torch.bfloat16)], -1)


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def values(packed, pairs, dtype=torch.float64):
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).to(dtype)
    parts = codes.unflatten(-1, (pairs.shape[-2], -1))
    return (parts * pairs[..., :1].to(dtype) + pairs[..., 1:].to(dtype)).flatten(-2)


def filled_cache(kernels, pages, kv_heads, page, head_dim, group, seed, device="cuda:0", spread=1.0):
    """A Kv4Cache whose every position holds quantised normal values (keys with loud channels)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    k = torch.randn((pages, kv_heads, page, head_dim), generator=gen, device=device) * spread
    k[..., :3] *= 4
    v = torch.randn((pages, kv_heads, page, head_dim), generator=gen, device=device) * spread
    kc, ks = quantise(k.to(torch.bfloat16), group)
    vc, vs = quantise(v.to(torch.bfloat16), group)
    return kernels.Kv4Cache(pack(kc), ks, pack(vc), vs)


def attend(q, cache, table, lengths, scale):
    """out, lse and the bound of the error of out, in 64 bits.

    A value is zero + scale * code; a weight times its scale is rounded to FP16 (2^-11), of at most
    15 of which each code takes, everything else is FP32.  A score is a sum of at most 128 products of
    exact FP16 numbers and of the zero's part: each of at most 128 + 8 additions rounds by 2^-24 of
    at most the sum of magnitudes, which moves a weight by as much (times two: numerator and
    denominator).  Exponentials, sums over the positions, rescalings and joins add a few 2^-22 more:
    2^-18 covers them.  All of that is relative to sum w (15 scale + |zero|).
    A weight times scale smaller than FP16's normal numbers is off by 2^-25 where the largest scale is
    more than 1/2 and the largest weight at least 2^7: less than length * 2^-27 of the largest scale.
    An exponential below FP32's smallest normal number, 2^-126 of one at the row's maximum, may come
    out as zero (so that a row whose heaviest value is exactly 0 has no smaller relative error):
    length * 2^-126 of the largest value, absolutely.
    Then the result is rounded once (2^-8 of it)."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64, device=q.device)
    group = q.shape[1] // cache.kv_heads
    for b, length in enumerate(lengths):
        if length <= 0:
            continue
        pages = table[b, : -(-length // cache.page)].long()
        for h in range(cache.kv_heads):
            k = values(cache.k_codes[pages, h].flatten(0, 1)[:length], cache.k_scales[pages, h].flatten(0, 1)[:length])
            v = values(cache.v_codes[pages, h].flatten(0, 1)[:length], cache.v_scales[pages, h].flatten(0, 1)[:length])
            heads = slice(h * group, (h + 1) * group)
            qh = q[b, heads].double()
            scores = qh @ k.T * scale
            pairs = cache.k_scales[pages, h].flatten(0, 1)[:length].double()
            size = (15 * pairs[..., 0].abs() + pairs[..., 1].abs()).amax()
            moved = 2 * 136 * 2.0 ** -24 * abs(scale) * qh.abs().sum(1, keepdim=True) * size + 2.0 ** -18
            w = torch.softmax(scores, -1)
            out[b, heads] = w @ v
            pairs = cache.v_scales[pages, h].flatten(0, 1)[:length].double()
            reach = (15 * pairs[..., 0].abs() + pairs[..., 1].abs()).repeat_interleave(cache.group, 1)
            bound[b, heads] = ((2.0 ** -11 + moved) * (w @ reach) + length * 2.0 ** -27 * pairs[..., 0].abs().amax()
                               + length * 2.0 ** -126 * v.abs().amax())
            lse[b, heads] = torch.logsumexp(scores, -1)
    return out, lse, bound + 2.0 ** -8 * (out.abs() + bound)


def scattered_table(lengths, page, spare, seed, device="cuda:0"):
    """A table of distinct pages in random order, unused entries far outside the cache."""
    held = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), max(1, max(held))), 2 ** 30, dtype=torch.int32)
    for row, count in enumerate(held):
        table[row, :count] = torch.tensor([order.pop() for _ in range(count)], dtype=torch.int32)
    return table.to(device), pages, order
