"""The operators of a served decoder layer, as they are measured.

Four groups, in the order in which one step of a layer uses them:

* ``norm``      a block's output normalised, gated and added to the scaled residual stream, and the
                normalised input of the next block (``kernels.rmsnorm_residual``);
* ``adapters``  a projection that all requests share plus a low-rank adapter for each row
                (``kernels.gemm_adapters``);
* ``cache``     new tokens written into a paged cache held in 4 bits and read back
                (``kernels.kv4_append``, ``kernels.kv4_read``);
* ``attend``    attention of one new token per sequence over that cache (``kernels.kv4_decode``).

``run`` computes them with elementary torch operations, or through the package where ``own`` is true.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _kernels():
    package = str(Path(__file__).resolve().parents[1] / "trinity-be_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from trinity_lowering import kernels
    return kernels


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of 16 sequences: the residual stream kept in FP32, a learned gate per column
        {"name": "norm_step_16x8192", "op": "norm", "rows": 16, "cols": 8192, "x": "bf16", "residual": "fp32",
         "gate": "column", "post": True, "scale": 1.0},
        # a long prompt or a large batch of prompts, BF16 throughout, norms on both sides of the block
        {"name": "norm_prompt_32768x4096", "op": "norm", "rows": 32768, "cols": 4096, "x": "bf16",
         "residual": "bf16", "gate": "none", "post": True, "scale": 1.0},
        # ragged sizes: an FP32 block output, a gate for every element, the residual damped
        {"name": "norm_ragged_5003x2055", "op": "norm", "rows": 5003, "cols": 2055, "x": "fp32",
         "residual": "bf16", "gate": "full", "post": False, "scale": 0.75},
        # the attention output projection of one decode step, requests with 12 different adapters
        {"name": "adapters_step_16x8192x8192_r16", "op": "adapters", "m": 16, "k": 8192, "n": 8192, "rank": 16,
         "adapters": 12, "segments": False},
        # a wide projection of an odd number of requests, higher rank, more adapters than fit one block
        {"name": "adapters_step_61x4096x28672_r64", "op": "adapters", "m": 61, "k": 4096, "n": 28672, "rank": 64,
         "adapters": 24, "segments": False},
        # prompts of several requests packed one behind the other
        {"name": "adapters_prompt_8192x8192x8192_r32", "op": "adapters", "m": 8192, "k": 8192, "n": 8192,
         "rank": 32, "adapters": 9, "segments": True},
        # one decode step: one token of each of 64 sequences
        {"name": "cache_step_64x8x128", "op": "cache", "tokens": 64, "kv_heads": 8, "head_dim": 128, "group": 64,
         "page": 64},
        # packed prompts of an odd total length
        {"name": "cache_prompt_32771x8x128", "op": "cache", "tokens": 32771, "kv_heads": 8, "head_dim": 128,
         "group": 32, "page": 64},
        # a single user: latency
        {"name": "attend_1x32x8_1023", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "group": 128, "page": 64, "length": 1023, "ragged": False},
        # a full decode batch
        {"name": "attend_64x64x8_4096", "op": "attend", "batch": 64, "heads": 64, "kv_heads": 8, "head_dim": 128,
         "group": 128, "page": 64, "length": 4096, "ragged": False},
        # many sequences of very different lengths (some empty), narrow heads, small pages and groups
        {"name": "attend_200x16x2_ragged", "op": "attend", "batch": 200, "heads": 16, "kv_heads": 2, "head_dim": 64,
         "group": 32, "page": 16, "length": 8191, "ragged": True},
        # two very long contexts, sixteen query heads for each cached head
        {"name": "attend_2x128x8_262144", "op": "attend", "batch": 2, "heads": 128, "kv_heads": 8, "head_dim": 128,
         "group": 64, "page": 128, "length": 262144, "ragged": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "adapters", "cache", "attend", "attend"])
    if op == "norm":
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = max(8, cols // 8 * 8)
        rows = _log(rng, 1, max(1, (32768 * 4096) // (2 * cols)))
        return {"op": op, "rows": rows, "cols": cols, "x": rng.choice(["bf16", "bf16", "fp32"]),
                "residual": rng.choice(["bf16", "fp32"]), "gate": rng.choice(["none", "column", "row", "full"]),
                "post": rng.random() < 0.6, "scale": rng.choice([1.0, 0.5, 0.75])}
    if op == "adapters":
        k = 8 * _log(rng, 32, 1024)
        n = 8 * _log(rng, 32, 2048)
        m = _log(rng, 1, 4096)
        return {"op": op, "m": m, "k": k, "n": n, "rank": 8 * rng.choice([1, 1, 2, 2, 3, 4, 6, 8, 16]),
                "adapters": _log(rng, 1, 32), "segments": m > 128 or rng.random() < 0.2}
    head_dim = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= head_dim])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "cache":
        return {"op": op, "tokens": _log(rng, 1, 16384), "kv_heads": kv_heads, "head_dim": head_dim, "group": group,
                "page": page}
    batch = _log(rng, 1, 256)
    length = _log(rng, 1, min(131072, (1 << 21) // (batch * kv_heads)))
    return {"op": op, "batch": batch, "heads": kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16, 24]),
            "kv_heads": kv_heads, "head_dim": head_dim, "group": group, "page": page, "length": length,
            "ragged": rng.random() < 0.6}


# ------------------------------------------------------------------------------------- inputs

def _randn(gen, shape, dtype=torch.bfloat16, factor=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)
    return x if factor == 1.0 else x * factor


def _adapter_rows(case):
    """Adapter of each row before the seed shuffles them: one row in five has none."""
    m, adapters = case["m"], case["adapters"]
    if not case["segments"]:
        return [-1 if i % 5 == 4 else i % adapters for i in range(m)]
    rng = random.Random(m * 31 + adapters)
    cuts = sorted(rng.randrange(m) for _ in range(adapters))
    rows, which = [], -1
    for i in range(m):
        while cuts and cuts[0] <= i:
            cuts.pop(0)
            which += 1
        rows.append(which)
    return rows


def _lengths(case):
    if not case["ragged"]:
        return [case["length"]] * case["batch"]
    rng = random.Random(case["batch"] * 131071 + case["length"])
    lengths = [_log(rng, 1, case["length"]) for _ in range(case["batch"])]
    for i in range(7, len(lengths), 16):
        lengths[i] = 0                       # a slot of the batch that no request holds
    lengths[0] = case["length"]
    return lengths


def _empty_cache(pages, case):
    kv_heads, page, head_dim = case["kv_heads"], case["page"], case["head_dim"]
    codes = [torch.zeros((pages, kv_heads, page, head_dim // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, kv_heads, page, head_dim // case["group"], 2), dtype=torch.bfloat16, device="cuda")
              for _ in range(2)]
    return {"k_codes": codes[0], "k_scales": scales[0], "v_codes": codes[1], "v_scales": scales[1]}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    op = case["op"]
    if op == "norm":
        rows, cols = case["rows"], case["cols"]
        state["x"] = _randn(gen, (rows, cols), _DTYPES[case["x"]])
        state["residual"] = _randn(gen, (rows, cols), _DTYPES[case["residual"]], 2.0)
        state["gain"] = 1.0 + _randn(gen, (cols,), torch.bfloat16, 0.25)
        state["post_gain"] = 1.0 + _randn(gen, (cols,), torch.bfloat16, 0.25) if case["post"] else None
        shape = {"none": None, "column": (1, cols), "row": (rows, 1), "full": (rows, cols)}[case["gate"]]
        state["gate"] = None if shape is None else _randn(gen, shape, torch.bfloat16, 0.5).expand(rows, cols)
        return state
    if op == "adapters":
        m, k, n, rank, adapters = (case[key] for key in ("m", "k", "n", "rank", "adapters"))
        state["x"] = _randn(gen, (m, k))
        state["w"] = _randn(gen, (k, n), factor=k ** -0.5)
        state["down"] = _randn(gen, (adapters, k, rank), factor=k ** -0.5)
        state["up"] = _randn(gen, (adapters, rank, n), factor=0.5 * rank ** -0.5)
        state["scales"] = 0.5 + torch.rand((adapters,), generator=gen, device="cuda")
        rows = _adapter_rows(case)
        if not case["segments"]:
            random.Random(seed).shuffle(rows)
        state["index"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        return state
    kv_heads, head_dim, page = case["kv_heads"], case["head_dim"], case["page"]
    # keys have a few loud channels in earnest
    loud = torch.ones((head_dim,), dtype=torch.bfloat16, device="cuda")
    loud[torch.randperm(head_dim, generator=gen, device="cuda")[:4]] = 4.0
    if op == "cache":
        tokens = case["tokens"]
        pages = -(-tokens // page) + 3
        state.update(_empty_cache(pages, case))
        # the two halves of one projection's output, as a program has them: views with a row pitch
        fused = _randn(gen, (tokens, 2, kv_heads, head_dim))
        fused[:, 0] *= loud
        state["k"], state["v"] = fused[:, 0], fused[:, 1]
        order = torch.randperm(pages, generator=gen, device="cuda")[: -(-tokens // page)]
        where = torch.arange(tokens, device="cuda")
        state["slots"] = order[where // page] * page + where % page
        return state
    lengths = _lengths(case)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + 2
    state.update(_empty_cache(pages, case))
    step = max(1, (1 << 25) // (kv_heads * page * head_dim))
    for first in range(0, pages, step):
        last = min(pages, first + step)
        for name in ("k", "v"):
            x = _randn(gen, (last - first, kv_heads, page, head_dim))
            if name == "k":
                x = x * loud
            codes, scales = _quantise(x.float(), case["group"])
            state[name + "_codes"][first:last] = _pack(codes)
            state[name + "_scales"][first:last] = scales
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table = torch.zeros((len(lengths), max(1, max(held))), dtype=torch.int32)
    for row, count in enumerate(held):
        table[row, :count] = torch.tensor([order.pop() for _ in range(count)], dtype=torch.int32)
    state["table"] = table.cuda()
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state["q"] = _randn(gen, (len(lengths), case["heads"], head_dim))
    state["scale"] = head_dim ** -0.5
    return state


# ------------------------------------------------------------------------------------- plain forms

def _quantise(x, group):
    """4-bit codes [..., D] and (scale, zero) pairs [..., D / group, 2] of FP32 values [..., D]."""
    parts = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    low, high = parts.amin(-1, keepdim=True), parts.amax(-1, keepdim=True)
    scale = ((high - low) / 15.0).to(torch.bfloat16).float()
    codes = torch.where(scale > 0, torch.round((parts - low) / scale).clamp(0.0, 15.0), torch.zeros_like(parts))
    return codes.to(torch.uint8).reshape(x.shape), torch.cat([scale, low], -1).to(torch.bfloat16)


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(packed, scales, dtype=torch.float32):
    """What packed codes [..., D / 2] with pairs [..., D / group, 2] stand for: [..., D]."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).to(dtype)
    groups = scales.shape[-2]
    parts = codes.reshape(*codes.shape[:-1], groups, codes.shape[-1] // groups)
    pairs = scales.to(dtype)
    return (parts * pairs[..., 0:1] + pairs[..., 1:2]).reshape(codes.shape)


def _plain_norm(s):
    case = s["case"]
    branch = s["x"].float()
    if case["post"]:
        branch = branch / torch.sqrt((branch * branch).mean(-1, keepdim=True) + 1e-6) * s["post_gain"].float()
    if s["gate"] is not None:
        branch = branch * s["gate"].float()
    h = s["residual"].float() * case["scale"] + branch
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * s["gain"].float()
    return h.to(s["residual"].dtype), y.to(torch.bfloat16)


def _plain_adapters(s):
    x = s["x"].float()
    out = x @ s["w"].float()
    for a in range(s["down"].shape[0]):
        delta = (x @ s["down"][a].float()) @ s["up"][a].float() * s["scales"][a]
        out = torch.where((s["index"] == a)[:, None], out + delta, out)
    return out.to(torch.bfloat16)


def _plain_cache(s):
    case, slots = s["case"], s["slots"]
    page, offset = slots // case["page"], slots % case["page"]
    result = []
    for name in ("k", "v"):
        codes, scales = _quantise(s[name].float(), case["group"])
        s[name + "_codes"][page, :, offset] = _pack(codes)
        s[name + "_scales"][page, :, offset] = scales
        result.append(_values(s[name + "_codes"][page, :, offset], s[name + "_scales"][page, :, offset]))
    return tuple(r.to(torch.bfloat16) for r in result)


def _plain_attend(s):
    case = s["case"]
    batch, heads, head_dim = s["q"].shape
    kv_heads = case["kv_heads"]
    table = s["table"].long()

    def gathered(name):
        codes = s[name + "_codes"][table].transpose(1, 2).flatten(2, 3)      # [batch, kv_heads, positions, D / 2]
        scales = s[name + "_scales"][table].transpose(1, 2).flatten(2, 3)
        return _values(codes, scales)

    q = s["q"].float().reshape(batch, kv_heads, heads // kv_heads, head_dim)
    scores = (q @ gathered("k").transpose(2, 3)) * s["scale"]
    live = torch.arange(scores.shape[-1], device="cuda") < s["lengths"][:, None]
    scores = torch.where(live[:, None, None, :], scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    out = (weights @ gathered("v")) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(batch, heads, head_dim).to(torch.bfloat16)


def _own_run(s):
    kernels = _kernels()
    case = s["case"]
    op = case["op"]
    if op == "norm":
        return kernels.rmsnorm_residual(s["x"], s["residual"], gain=s["gain"], post_gain=s["post_gain"],
                                        gate=s["gate"], residual_scale=case["scale"], eps=1e-6)
    if op == "adapters":
        return kernels.gemm_adapters(s["x"], s["w"], s["down"], s["up"], s["index"], scales=s["scales"])
    cache = kernels.Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    if op == "cache":
        kernels.kv4_append(cache, s["k"], s["v"], s["slots"])
        return kernels.kv4_read(cache, s["slots"])
    return kernels.kv4_decode(s["q"], cache, s["table"], s["lengths"], s["scale"])


def run(state):
    if own:
        return _own_run(state)
    return {"norm": _plain_norm, "adapters": _plain_adapters, "cache": _plain_cache,
            "attend": _plain_attend}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "norm":
        rows, cols = case["rows"], case["cols"]
        size = {"bf16": 2, "fp32": 4}
        gate = {"none": 0, "column": cols, "row": rows, "full": rows * cols}[case["gate"]]
        per = size[case["x"]] + 2 * size[case["residual"]] + 2
        return {"bytes": rows * cols * per + 2 * gate + 2 * cols * (2 if case["post"] else 1),
                "flops": rows * cols * (10 if case["post"] else 7)}
    if op == "adapters":
        m, k, n, rank = case["m"], case["k"], case["n"], case["rank"]
        rows = _adapter_rows(case)
        used = len(set(rows) - {-1})
        with_adapter = sum(1 for r in rows if r >= 0)
        return {"bytes": 2 * (m * k + k * n + m * n + used * rank * (k + n)) + 4 * m + 4 * used,
                "flops": 2 * m * k * n + 2 * with_adapter * rank * (k + n)}
    head_dim, kv_heads = case["head_dim"], case["kv_heads"]
    row = head_dim // 2 + 4 * (head_dim // case["group"])          # bytes of one cached key or value
    if op == "cache":
        rows = 2 * case["tokens"] * kv_heads
        return {"bytes": rows * (4 * head_dim + 2 * row) + 8 * case["tokens"], "flops": rows * head_dim * 7}
    lengths = _lengths(case)
    total = sum(lengths)
    used_pages = sum(-(-n // case["page"]) for n in lengths)
    return {"bytes": 2 * total * kv_heads * row + 4 * len(lengths) * case["heads"] * head_dim + 4 * used_pages
            + 4 * len(lengths),
            "flops": 4 * total * case["heads"] * head_dim}


# ------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op == "norm":
        x = s["x"].to(f64)
        if case["post"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s["post_gain"].to(f64)
        if s["gate"] is not None:
            x = x * s["gate"].to(f64)
        h = torch.add(x, s["residual"].to(f64), alpha=case["scale"])
        return h, h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s["gain"].to(f64)
    if op == "adapters":
        x = s["x"].to(f64)
        out = x @ s["w"].to(f64)
        for a, factor in enumerate(s["scales"].tolist()):
            rows = torch.nonzero(s["index"] == a).flatten()
            out[rows] += factor * (x[rows] @ s["down"][a].to(f64) @ s["up"][a].to(f64))
        return out
    if op == "cache":
        result = []
        for x in (s["k"], s["v"]):
            parts = x.to(f64).unflatten(-1, (-1, case["group"]))
            low = parts.min(-1, keepdim=True).values
            step = (parts.max(-1, keepdim=True).values - low).div(15).to(torch.bfloat16).to(f64)
            code = torch.nan_to_num((parts - low) / step).round().clamp(0, 15)
            result.append((low + step * code).flatten(-2))
        return tuple(result)
    outputs = []
    group = case["heads"] // case["kv_heads"]
    for b, length in enumerate(s["lengths"].tolist()):
        q = s["q"][b].to(f64)
        if length == 0:
            outputs.append(torch.zeros_like(q))
            continue
        pages = s["table"][b, : -(-length // case["page"])].long()
        heads = []
        for h in range(case["kv_heads"]):
            both = []
            for name in ("k", "v"):
                codes = s[name + "_codes"][pages, h].flatten(0, 1)[:length].to(torch.int32)
                pairs = s[name + "_scales"][pages, h].flatten(0, 1)[:length].to(f64).repeat_interleave(case["group"], 1)
                both.append(torch.stack((codes % 16, codes // 16), -1).flatten(1).to(f64) * pairs[..., 0]
                            + pairs[..., 1])
            logits = q[h * group:(h + 1) * group] @ both[0].T * s["scale"]
            heads.append(torch.softmax(logits, -1) @ both[1])
        outputs.append(torch.cat(heads))
    return torch.stack(outputs)
