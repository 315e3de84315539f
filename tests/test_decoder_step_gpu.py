"""The serving operators as they are used together: decode steps of one attention block with adapters, a
4-bit cache and fused seams, eagerly and as a replayed CUDA graph (B200 only)."""
import pytest
import torch

import kv4_reference as ref
import test_adapters_gpu as adapters_test
import test_block_norm_gpu as norm_test

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
D_MODEL, HEADS, KV_HEADS, HEAD_DIM, GROUP, PAGE = 1024, 16, 4, 128, 64, 32


@pytest.fixture(scope="module")
def kernels():
    from trinity_lowering import kernels as k
    k.library()
    return k


class Block:
    """Weights, cache and state of one block for a batch of sequences of different lengths."""

    def __init__(self, kernels, lengths, seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
        self.k, self.batch = kernels, len(lengths)
        width = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        self.w_qkv = (rand(D_MODEL, width) * D_MODEL ** -0.5).to(BF16)
        self.w_o = (rand(HEADS * HEAD_DIM, D_MODEL) * (HEADS * HEAD_DIM) ** -0.5).to(BF16)
        lora = lambda k, n, r: ((rand(3, k, r) * k ** -0.5).to(BF16), (rand(3, r, n) * 0.5 * r ** -0.5).to(BF16))
        self.a_qkv, self.a_o = lora(D_MODEL, width, 16), lora(HEADS * HEAD_DIM, D_MODEL, 8)
        self.index = torch.tensor([i % 4 - 1 for i in range(self.batch)], dtype=torch.int32, device=DEV)
        self.gains = [(1 + 0.1 * rand(D_MODEL)).to(BF16) for _ in range(3)]
        self.gate = (0.5 * rand(1, D_MODEL)).to(BF16)
        capacity = [n + 8 for n in lengths]
        self.table, pages, _ = ref.scattered_table(capacity, PAGE, 1, seed)
        self.table = torch.where(self.table < pages, self.table, torch.zeros_like(self.table))
        self.cache = ref.filled_cache(kernels, pages, KV_HEADS, PAGE, HEAD_DIM, GROUP, seed)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        self.branch, self.stream = rand(self.batch, D_MODEL).to(BF16), rand(self.batch, D_MODEL)

    def slots(self):
        """The place of each sequence's new token; sequences that have ended (length 0) have none."""
        at = self.lengths.long()
        page = self.table.gather(1, (at // PAGE)[:, None])[:, 0].long()
        return torch.where(at > 0, page * PAGE + at % PAGE, torch.full_like(at, -1))

    def step(self):
        """One token of every sequence; returns every intermediate result."""
        k = self.k
        h, x = k.rmsnorm_residual(self.branch, self.stream, gain=self.gains[0], post_gain=self.gains[1], eps=1e-6)
        qkv = k.gemm_adapters(x, self.w_qkv, *self.a_qkv, self.index)
        heads = qkv.unflatten(1, (HEADS + 2 * KV_HEADS, HEAD_DIM))
        q, new_k, new_v = heads.split((HEADS, KV_HEADS, KV_HEADS), 1)
        slots = self.slots()
        k.kv4_append(self.cache, new_k, new_v, slots)
        lengths = self.lengths + (self.lengths > 0)
        attended = k.kv4_decode(q, self.cache, self.table, lengths, HEAD_DIM ** -0.5)
        o = k.gemm_adapters(attended.flatten(1), self.w_o, *self.a_o, self.index)
        h2, y = k.rmsnorm_residual(o, h, gain=self.gains[2], gate=self.gate, residual_scale=0.9, eps=1e-6)
        return {"h": h, "x": x, "qkv": qkv, "slots": slots, "lengths": lengths, "attended": attended, "o": o, "h2": h2, "y": y}


def test_stages_of_a_step(kernels):
    """Every stage against 64 bits, from what the stage before it returned."""
    block = Block(kernels, [40, 1, 0, 130, 257, 31], 1)
    branch, stream = block.branch, block.stream
    s = block.step()
    norm_test.check(s["h"], s["x"], norm_test.formulas(branch, stream, block.gains[0], block.gains[1], None, 1.0, 1e-6, True),
                    block.gains[0])
    adapters_test.check(s["qkv"], *adapters_test.expected(s["x"], block.w_qkv, *block.a_qkv, block.index, None, None))
    heads = s["qkv"].unflatten(1, (HEADS + 2 * KV_HEADS, HEAD_DIM))
    kept = s["slots"] >= 0
    back = kernels.kv4_read(block.cache, s["slots"], dtype=torch.float32)
    for got, new in zip(back, heads[:, HEADS:].split(KV_HEADS, 1)):
        codes, pairs = ref.quantise(new[kept], GROUP)
        assert torch.equal(got[kept], ref.values(ref.pack(codes), pairs, torch.float32))
    want, _, bound = ref.attend(heads[:, :HEADS], block.cache, block.table, s["lengths"].tolist(), HEAD_DIM ** -0.5)
    assert ((s["attended"].double() - want).abs() <= bound).all()
    assert (s["attended"][2] == 0).all()
    adapters_test.check(s["o"], *adapters_test.expected(s["attended"].flatten(1), block.w_o, *block.a_o, block.index, None, None))
    norm_test.check(s["h2"], s["y"], norm_test.formulas(s["o"], s["h"], block.gains[2], None, block.gate, 0.9, 1e-6, False),
                    block.gains[2])


def test_replayed_steps_equal_eager_ones(kernels):
    """Six steps, each from the last one's result and lengths: a captured step, replayed, gives the bits of
    eager calls, cache included."""
    lengths = [33, 7, 0, 190, 64]
    eager, graphed = Block(kernels, lengths, 2), Block(kernels, lengths, 2)
    graphed.step()                     # warm-up outside the capture; its token is written again below
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = graphed.step()
    for _ in range(6):
        s = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for name, value in s.items():
            assert torch.equal(value, static[name]), name
        for block, out in ((eager, s), (graphed, static)):
            block.branch.copy_(out["y"])
            block.stream.copy_(out["h2"])
            block.lengths.copy_(out["lengths"])
    assert all(torch.equal(a, b) for a, b in zip(eager.cache.tensors, graphed.cache.tensors))
    assert kernels.device_status() == 0
