"""Refused layouts have a workspace of 0 bytes, which a binding passes on as a null pointer: the message names the
layout all the same (no GPU)."""
import ctypes

import pytest

from trinity_lowering import kernels as k

BASE = 1 << 24


def message(code, expected):
    assert code == expected
    return k.library().trinity_sm100_last_error().decode()


@pytest.mark.parametrize("changes,code,text", [
    ({"heads": 7}, -1, "divide"), ({"heads": 0}, -1, "empty"), ({"table_stride": 3}, -1, "table"), ({}, -1, "null workspace")])
def test_decode(changes, code, text):
    cache = k.Kv4CacheArgs(BASE, 2 * BASE, 3 * BASE, 4 * BASE, 8, 2, 32, 128, 64, 0)
    args = k.Kv4DecodeArgs(5 * BASE, 6 * BASE, 7 * BASE, 8 * BASE, None, None, 0, 1024, 128, 4, 3, 8, 4, 0.1)
    for name, value in changes.items():
        setattr(args, name, value)
    assert text in message(k.library().trinity_sm100_kv4_decode(ctypes.byref(cache), ctypes.byref(args), None), code)


@pytest.mark.parametrize("changes,code,text", [({"rank": 136, "ld_down": 136}, -2, "rank 136"), ({"rank": 12}, -2, "rank 12"),
                                               ({"count": 0}, -1, "no adapters"), ({}, -1, "null workspace")])
def test_adapters(changes, code, text):
    gemm = k.GemmArgs(BASE, 2 * BASE, None, None, 3 * BASE, 4, 64, 128, 128, 64, 64, 0, k.BIAS_NONE, k.ACT_NONE, k.DT_BF16, 0)
    args = k.AdaptersArgs(4 * BASE, 5 * BASE, 6 * BASE, None, None, 0, 16, 2048, 64, 1024, 3, 16)
    for name, value in changes.items():
        setattr(args, name, value)
    assert text in message(k.library().trinity_sm100_gemm_adapters_bf16(ctypes.byref(gemm), ctypes.byref(args), None), code)


def test_a_size_of_zero_is_not_kept(monkeypatch):
    """A query that failed must not decide what later calls allocate."""
    answers = [0, 4096]

    class Library:
        def trinity_sm100_kv4_decode_workspace_bytes(self, *layout):
            return answers.pop(0)

    monkeypatch.setattr(k, "library", lambda: Library())
    monkeypatch.setattr(k.torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(k, "_kv4_workspaces", {})
    assert [k.kv4_decode_workspace_bytes(8, 2, 128) for _ in range(3)] == [0, 4096, 4096]
