"""Refusals of the adapter and 4-bit cache entry points (no GPU: argument checks come before any device
call), and of their bindings for host tensors."""
import ctypes

import pytest
import torch

from trinity_lowering import kernels as k

BASE = 1 << 24


def cache(**changes):
    args = k.Kv4CacheArgs(BASE, 2 * BASE, 3 * BASE, 4 * BASE, 8, 2, 32, 128, 64, 0)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


def rows(**changes):
    args = k.Kv4RowsArgs(5 * BASE, 6 * BASE, 7 * BASE, 3, 256, 128, 256, 128)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


def decode(**changes):
    args = k.Kv4DecodeArgs(5 * BASE, 6 * BASE, 7 * BASE, 8 * BASE, None, 9 * BASE, 1 << 30, 1024, 128, 4, 3, 8, 4, 0.1)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


BAD_CACHES = [({"k_codes": None}, -1), ({"v_scales": None}, -1), ({"k_codes": BASE + 8}, -1), ({"head_dim": 96}, -2),
              ({"head_dim": 256}, -2), ({"group": 16}, -2), ({"group": 96}, -2), ({"head_dim": 64, "group": 128}, -2),
              ({"pages": 0}, -1), ({"kv_heads": -1}, -1), ({"page": 0}, -1), ({"page": 24}, -2),
              ({"pages": 1 << 20, "kv_heads": 128}, -2)]


@pytest.mark.parametrize("changes,code", BAD_CACHES)
def test_caches(changes, code):
    lib = k.library()
    c = ctypes.byref(cache(**changes))
    assert lib.trinity_sm100_kv4_append(c, ctypes.byref(rows()), None) == code
    assert lib.trinity_sm100_kv4_read(c, ctypes.byref(rows()), k.DT_BF16, None) == code
    assert lib.trinity_sm100_kv4_decode(c, ctypes.byref(decode()), None) == code
    assert b"kv4" in lib.trinity_sm100_last_error()


@pytest.mark.parametrize("changes,code", [({"k": None}, -1), ({"slots": None}, -1), ({"tokens": 0}, -1), ({"tokens": 1 << 40}, -2),
                                          ({"slots": 7 * BASE + 4}, -1)])
def test_rows(changes, code):
    lib = k.library()
    for call in (lambda r: lib.trinity_sm100_kv4_append(ctypes.byref(cache()), r, None),
                 lambda r: lib.trinity_sm100_kv4_read(ctypes.byref(cache()), r, k.DT_BF16, None)):
        assert call(ctypes.byref(rows(**changes))) == code
    assert lib.trinity_sm100_kv4_append(ctypes.byref(cache()), ctypes.byref(rows(k=5 * BASE + 1)), None) == -1
    for changes in ({"k": 5 * BASE + 8}, {"v_token_stride": 260}):
        assert lib.trinity_sm100_kv4_read(ctypes.byref(cache()), ctypes.byref(rows(**changes)), k.DT_BF16, None) == -1
    assert lib.trinity_sm100_kv4_read(ctypes.byref(cache()), ctypes.byref(rows()), 5, None) == -1


@pytest.mark.parametrize("changes,code,text", [
    ({"q": None}, -1, "null"), ({"workspace": None}, -1, "null"), ({"batch": 0}, -1, "empty"), ({"max_pages": 0}, -1, "empty"),
    ({"heads": 7}, -1, "divide"), ({"table_stride": 3}, -1, "table"), ({"q": 5 * BASE + 2}, -1, "16 bytes"),
    ({"q_head_stride": 130}, -1, "16 bytes"), ({"out": 8 * BASE + 8}, -1, "aligned"), ({"lengths": 7 * BASE + 2}, -1, "aligned"),
    ({"max_pages": 1 << 27, "table_stride": 1 << 27}, -2, "2^31"),
    ({"max_pages": 1 << 25, "table_stride": 1 << 25, "heads": 1 << 14}, -2, "too long")])
def test_decode(changes, code, text):
    lib = k.library()
    assert lib.trinity_sm100_kv4_decode(ctypes.byref(cache()), ctypes.byref(decode(**changes)), None) == code
    assert text in lib.trinity_sm100_last_error().decode()


def test_null_blocks():
    lib = k.library()
    assert lib.trinity_sm100_kv4_append(None, None, None) == -1
    assert lib.trinity_sm100_kv4_read(ctypes.byref(cache()), None, 0, None) == -1
    assert lib.trinity_sm100_kv4_decode(None, ctypes.byref(decode()), None) == -1
    assert lib.trinity_sm100_gemm_adapters_bf16(None, None, None) == -1


def gemm(**changes):
    args = k.GemmArgs(BASE, 2 * BASE, None, None, 3 * BASE, 4, 64, 128, 128, 64, 64, 0, k.BIAS_NONE, k.ACT_NONE, k.DT_BF16, 0)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


def adapters(**changes):
    args = k.AdaptersArgs(4 * BASE, 5 * BASE, 6 * BASE, None, 7 * BASE, 1 << 30, 16, 2048, 64, 1024, 3, 16)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("g,a,code", [
    ({"a": None}, {}, -1), ({"m": 0}, {}, -1), ({"lda": 100}, {}, -1), ({"activation": k.ACT_SILU_GATE, "b2": BASE}, {}, -2),
    ({"bias_mode": k.BIAS_ROW_VECTOR, "bias": BASE}, {}, -2), ({"bias_mode": k.BIAS_MATRIX, "bias": BASE, "ld_bias": 64}, {}, -2),
    ({"k": 124}, {}, -2), ({"n": 60}, {}, -2), ({"m": 1 << 21}, {}, -2),
    ({}, {"down": None}, -1), ({}, {"index": None}, -1), ({}, {"workspace": None}, -1), ({}, {"count": 0}, -1),
    ({}, {"rank": 0}, -2), ({}, {"rank": 12}, -2), ({}, {"rank": 136}, -2), ({}, {"ld_down": 8}, -1), ({}, {"ld_up": 56}, -1),
    ({}, {"ld_up": 68}, -1), ({}, {"down": 4 * BASE + 8}, -1), ({}, {"stride_up": 0}, -1), ({}, {"stride_down": -2048}, -1),
    ({}, {"index": 6 * BASE + 2}, -1), ({}, {"workspace_bytes": 10}, -1)])
def test_adapters(g, a, code):
    lib = k.library()
    assert lib.trinity_sm100_gemm_adapters_bf16(ctypes.byref(gemm(**g)), ctypes.byref(adapters(**a)), None) == code


def test_workspace_sizes():
    assert k.gemm_adapters_workspace_bytes(16, 8192, 16) >= 16 * (16 + 8192) * 2
    assert k.gemm_adapters_workspace_bytes(0, 8192, 16) == 0 and k.gemm_adapters_workspace_bytes(16, 8, 256) == 0


def test_bindings_refuse_host_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        k.kv4_cache(2, 1, 16, 64, 32, "cpu")
    with pytest.raises(ValueError):
        k.gemm_adapters(x, x.t().contiguous(), x[None, :, :8], x[None, :8], torch.zeros(4, dtype=torch.int32))
