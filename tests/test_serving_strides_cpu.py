"""The stride of an axis with one entry has no meaning and refuses no call (no GPU: each call is ended by a check
that comes later)."""
import ctypes

import torch

from trinity_lowering import kernels as k

BASE = 1 << 24


def test_pitch_of_one_row():
    wide = torch.zeros(3, 267)
    assert k._pitch(wide[1:2, :264]) == 264 and k._pitch(wide[:, :264]) == 267 and k._pitch(wide[:1]) == 267
    assert k._pitch(wide[:1, :264].expand(3, 264)) == 0


def test_decode():
    cache = k.Kv4CacheArgs(BASE, 2 * BASE, 3 * BASE, 4 * BASE, 8, 1, 32, 128, 64, 0)

    def answer(batch, heads, batch_stride, head_stride):
        args = k.Kv4DecodeArgs(5 * BASE, 6 * BASE, 7 * BASE, 8 * BASE + 8, None, 9 * BASE, 1 << 30, batch_stride, head_stride, 4,
                               batch, heads, 4, 0.1)
        assert k.library().trinity_sm100_kv4_decode(ctypes.byref(cache), ctypes.byref(args), None) == -1
        return k.library().trinity_sm100_last_error().decode()

    assert "pointers must be" in answer(1, 4, 1027, 128)
    assert "pointers must be" in answer(3, 1, 1024, 131)
    assert "query rows" in answer(2, 4, 1027, 128) and "query rows" in answer(1, 4, 1024, 131)


def test_adapters():
    gemm = k.GemmArgs(BASE, 2 * BASE, None, None, 3 * BASE, 1 << 21, 64, 128, 128, 64, 64, 0, k.BIAS_NONE, k.ACT_NONE, k.DT_BF16, 0)
    for count, text in ((1, "too many rows"), (2, "16 bytes")):
        args = k.AdaptersArgs(4 * BASE, 5 * BASE, 6 * BASE, None, 7 * BASE, 1 << 40, 16, 2051, 64, 1027, count, 16)
        assert k.library().trinity_sm100_gemm_adapters_bf16(ctypes.byref(gemm), ctypes.byref(args), None) != 0
        assert text in k.library().trinity_sm100_last_error().decode()
