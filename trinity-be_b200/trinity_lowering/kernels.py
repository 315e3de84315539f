"""ctypes binding of the sm_100a kernel library (``include/trinity_sm100.h``).

This is the only route from Python to the CUDA kernels.  There is no CPU or PyTorch
fallback: when the shared library is missing or a call fails, an exception is raised.
PyTorch tensors are used for device memory and streams only; the C ABI sees raw pointers.
"""
import ctypes
import threading
from pathlib import Path

import torch

_LIB_PATH = Path(__file__).resolve().parents[1] / "lib" / "libtrinity_sm100.so"

BIAS_NONE, BIAS_COL_VECTOR, BIAS_ROW_VECTOR, BIAS_MATRIX = 0, 1, 2, 3
ACT_NONE, ACT_RELU, ACT_SILU, ACT_SILU_GATE = 0, 1, 2, 3
DT_BF16, DT_FP32 = 0, 1

EXPORTS = (
    "trinity_sm100_gemm_bf16",
    "trinity_sm100_gemm_batched_bf16",
    "trinity_sm100_gemm_adapters_workspace_bytes",
    "trinity_sm100_gemm_adapters_bf16",
    "trinity_sm100_gemm_pair_capacity",
    "trinity_sm100_rmsnorm_bf16",
    "trinity_sm100_rmsnorm_residual",
    "trinity_sm100_softmax_bf16",
    "trinity_sm100_mla_scratch_bytes",
    "trinity_sm100_mla_default_splits",
    "trinity_sm100_mla_balanced_slots",
    "trinity_sm100_mla_schedule",
    "trinity_sm100_mla_schedule_segment",
    "trinity_sm100_mla_decode_bf16",
    "trinity_sm100_mla_decode_bf16_noalloc",
    "trinity_sm100_kv4_append",
    "trinity_sm100_kv4_read",
    "trinity_sm100_kv4_decode_workspace_bytes",
    "trinity_sm100_kv4_decode",
    "trinity_sm100_allreduce_flag_words",
    "trinity_sm100_allreduce_bf16",
    "trinity_sm100_allgather_bf16",
    "trinity_sm100_gemm_allreduce_flag_words",
    "trinity_sm100_gemm_allreduce_bf16",
    "trinity_sm100_gemm_allreduce_stamps",
    "trinity_sm100_gemm_allreduce_workspace_bytes",
    "trinity_sm100_gemm_allreduce_workspace_bf16",
    "trinity_sm100_pointwise",
    "trinity_sm100_row_reduce_sum",
    "trinity_sm100_prepare_device",
    "trinity_sm100_current_device",
    "trinity_sm100_stream_synchronize",
    "trinity_sm100_device_status",
    "trinity_sm100_set_wait_budget",
    "trinity_sm100_abi_version",
    "trinity_sm100_last_error",
    "trinity_sm100_launch_count",
)


class KernelError(RuntimeError):
    """A kernel-library call returned a non-zero code."""

    def __init__(self, code, message):
        super().__init__(f"trinity_sm100 error {code}: {message}")
        self.code = code


class GemmArgs(ctypes.Structure):
    _fields_ = [
        ("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("b2", ctypes.c_void_p),
        ("bias", ctypes.c_void_p), ("out", ctypes.c_void_p),
        ("m", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64),
        ("lda", ctypes.c_int64), ("ldb", ctypes.c_int64), ("ldo", ctypes.c_int64),
        ("ld_bias", ctypes.c_int64),
        ("bias_mode", ctypes.c_int32), ("activation", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32), ("reserved", ctypes.c_int32),
    ]


class GemmBatchArgs(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int64), ("stride_a", ctypes.c_int64), ("stride_b", ctypes.c_int64),
                ("stride_out", ctypes.c_int64), ("stride_bias", ctypes.c_int64)]


class AdaptersArgs(ctypes.Structure):
    _fields_ = [
        ("down", ctypes.c_void_p), ("up", ctypes.c_void_p), ("index", ctypes.c_void_p),
        ("scales", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
        ("ld_down", ctypes.c_int64), ("stride_down", ctypes.c_int64),
        ("ld_up", ctypes.c_int64), ("stride_up", ctypes.c_int64),
        ("count", ctypes.c_int32), ("rank", ctypes.c_int32),
    ]


class RmsnormResidualArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("gate", ctypes.c_void_p),
        ("gain", ctypes.c_void_p), ("post_gain", ctypes.c_void_p),
        ("residual_out", ctypes.c_void_p), ("out", ctypes.c_void_p),
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
        ("ld_x", ctypes.c_int64), ("ld_residual", ctypes.c_int64),
        ("ld_residual_out", ctypes.c_int64), ("ld_out", ctypes.c_int64),
        ("gate_row_stride", ctypes.c_int64), ("gate_col_stride", ctypes.c_int64),
        ("x_dtype", ctypes.c_int32), ("residual_dtype", ctypes.c_int32),
        ("post_norm", ctypes.c_int32), ("eps", ctypes.c_float), ("post_eps", ctypes.c_float),
        ("residual_scale", ctypes.c_float),
    ]


class MlaArgs(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p), ("cache", ctypes.c_void_p), ("out", ctypes.c_void_p),
        ("scratch", ctypes.c_void_p), ("scratch_bytes", ctypes.c_size_t),
        ("batch", ctypes.c_int32), ("heads", ctypes.c_int32), ("seq", ctypes.c_int32),
        ("d_qk", ctypes.c_int32), ("d_v", ctypes.c_int32), ("kv_splits", ctypes.c_int32),
        ("scale", ctypes.c_float), ("reserved", ctypes.c_int32),
    ]


class Kv4CacheArgs(ctypes.Structure):
    _fields_ = [
        ("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p),
        ("v_codes", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
        ("pages", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("page", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("group", ctypes.c_int32), ("reserved", ctypes.c_int32),
    ]


class Kv4RowsArgs(ctypes.Structure):
    _fields_ = [
        ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("slots", ctypes.c_void_p),
        ("tokens", ctypes.c_int64),
        ("k_token_stride", ctypes.c_int64), ("k_head_stride", ctypes.c_int64),
        ("v_token_stride", ctypes.c_int64), ("v_head_stride", ctypes.c_int64),
    ]


class Kv4DecodeArgs(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("lengths", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("q_batch_stride", ctypes.c_int64), ("q_head_stride", ctypes.c_int64),
        ("table_stride", ctypes.c_int64),
        ("batch", ctypes.c_int32), ("heads", ctypes.c_int32), ("max_pages", ctypes.c_int32),
        ("scale", ctypes.c_float),
    ]


class AllReduceArgs(ctypes.Structure):
    _fields_ = [
        ("peers", ctypes.POINTER(ctypes.c_void_p)), ("flags", ctypes.POINTER(ctypes.c_void_p)),
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
        ("world", ctypes.c_int32), ("rank", ctypes.c_int32),
        ("epoch", ctypes.c_uint32), ("reserved", ctypes.c_int32),
    ]


_lock = threading.Lock()
_lib = None


def library_path():
    return _LIB_PATH


def library():
    """Loads the kernel library once; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not _LIB_PATH.exists():
                raise RuntimeError(
                    f"{_LIB_PATH} is missing: build it with `python -m __graft_entry__` "
                    "(there is no fallback path)")
            lib = ctypes.CDLL(str(_LIB_PATH))
            lib.trinity_sm100_gemm_bf16.argtypes = [ctypes.POINTER(GemmArgs), ctypes.c_void_p]
            lib.trinity_sm100_gemm_adapters_workspace_bytes.argtypes = [
                ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]
            lib.trinity_sm100_gemm_adapters_workspace_bytes.restype = ctypes.c_size_t
            lib.trinity_sm100_gemm_adapters_bf16.argtypes = [
                ctypes.POINTER(GemmArgs), ctypes.POINTER(AdaptersArgs), ctypes.c_void_p]
            lib.trinity_sm100_rmsnorm_bf16.argtypes = [
                ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64,
                ctypes.c_float, ctypes.c_void_p]
            lib.trinity_sm100_rmsnorm_residual.argtypes = [
                ctypes.POINTER(RmsnormResidualArgs), ctypes.c_void_p]
            lib.trinity_sm100_softmax_bf16.argtypes = [
                ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p]
            lib.trinity_sm100_mla_scratch_bytes.argtypes = [ctypes.c_int32] * 4
            lib.trinity_sm100_mla_scratch_bytes.restype = ctypes.c_size_t
            lib.trinity_sm100_mla_default_splits.argtypes = [ctypes.c_int32] * 2
            lib.trinity_sm100_mla_balanced_slots.argtypes = [ctypes.c_int32] * 2
            lib.trinity_sm100_mla_decode_bf16.argtypes = [ctypes.POINTER(MlaArgs), ctypes.c_void_p]
            lib.trinity_sm100_mla_decode_bf16_noalloc.argtypes = [
                ctypes.POINTER(MlaArgs), ctypes.c_void_p]
            lib.trinity_sm100_kv4_append.argtypes = [
                ctypes.POINTER(Kv4CacheArgs), ctypes.POINTER(Kv4RowsArgs), ctypes.c_void_p]
            lib.trinity_sm100_kv4_read.argtypes = [
                ctypes.POINTER(Kv4CacheArgs), ctypes.POINTER(Kv4RowsArgs), ctypes.c_int32, ctypes.c_void_p]
            lib.trinity_sm100_kv4_decode_workspace_bytes.argtypes = [ctypes.c_int32] * 3
            lib.trinity_sm100_kv4_decode_workspace_bytes.restype = ctypes.c_size_t
            lib.trinity_sm100_kv4_decode.argtypes = [
                ctypes.POINTER(Kv4CacheArgs), ctypes.POINTER(Kv4DecodeArgs), ctypes.c_void_p]
            lib.trinity_sm100_allreduce_flag_words.restype = ctypes.c_size_t
            lib.trinity_sm100_allreduce_bf16.argtypes = [
                ctypes.POINTER(AllReduceArgs), ctypes.c_void_p]
            lib.trinity_sm100_allgather_bf16.argtypes = [
                ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64,
                ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]
            lib.trinity_sm100_gemm_allreduce_flag_words.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]
            lib.trinity_sm100_gemm_allreduce_flag_words.restype = ctypes.c_size_t
            lib.trinity_sm100_gemm_allreduce_bf16.argtypes = [
                ctypes.POINTER(GemmArgs), ctypes.POINTER(AllReduceArgs), ctypes.c_void_p]
            lib.trinity_sm100_device_status.argtypes = [
                ctypes.POINTER(ctypes.c_uint32), ctypes.c_int]
            lib.trinity_sm100_set_wait_budget.argtypes = [ctypes.c_uint64]
            lib.trinity_sm100_last_error.restype = ctypes.c_char_p
            lib.trinity_sm100_launch_count.restype = ctypes.c_uint64
            _lib = lib
    return _lib


def _check(code):
    if code != 0:
        raise KernelError(code, library().trinity_sm100_last_error().decode())


def _stream(stream=None):
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _require(t, dtype, name):
    if not t.is_cuda or t.dtype != dtype:
        raise ValueError(f"{name}: expected a CUDA tensor of {dtype}, got {t.device} {t.dtype}")


def _submit(device, stream, operands, launch):
    """``launch(handle)`` with ``device`` current and ``handle`` the stream to launch on.

    Memory that ``launch`` allocates (outputs, scratch) belongs to that stream.  On a stream other
    than the device's current one the allocator is told that the operands are in use there and the
    results here, so neither is handed out again too early; ordering the two streams is left to
    the caller, as with every torch operation."""
    if stream is None:
        index = device.index
        if index == torch._C._cuda_getDevice():     # the common case, a few hundred nanoseconds
            return launch(torch._C._cuda_getCurrentRawStream(index))
        with torch.cuda.device(device):
            return launch(torch.cuda.current_stream().cuda_stream)
    if stream.device != device:
        raise ValueError(f"the stream belongs to {stream.device}, the operands to {device}")
    with torch.cuda.device(device):
        here = torch.cuda.current_stream()
        if stream == here:
            return launch(here.cuda_stream)
        with torch.cuda.stream(stream):
            result = launch(stream.cuda_stream)
        for t in operands:
            if t is not None:
                t.record_stream(stream)
        for t in result if isinstance(result, tuple) else (result,):
            if t is not None:
                t.record_stream(here)
        return result


def _operand(t, dtype, index, name):
    """Checks the type of an operand and that it lies on CUDA device ``index``."""
    if t.dtype != dtype or t.get_device() != index or index < 0:
        raise ValueError(f"{name}: expected a tensor of {dtype} on cuda:{max(index, 0)}, got {t.device} {t.dtype}")


def _workspace_operand(t, index, what):
    """A workspace of any type; the kernels write its ``numel() * element_size()`` bytes from its first on."""
    if t.get_device() != index:
        raise ValueError(f"{what}: the workspace is on another device")
    if not t.is_contiguous():
        raise ValueError(f"{what}: the workspace must be contiguous")


def _rows_ok(t):
    """A [rows, cols] tensor with a unit inner stride (of no meaning when there is one column)."""
    return t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1)


def _pitch(t):
    """Row pitch of a [rows, cols] tensor in elements (a single row has none that means anything: its width)."""
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else cols


def _empty_rows(like, dtype):
    """An uninitialised contiguous tensor of ``like``'s shape (empty_like is the cheaper call)."""
    if like.dtype is dtype and like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty(like.shape, dtype=dtype, device=like.device)


def _real_operand(t, index, name):
    """``_operand`` for either of BF16 and FP32; the type's code."""
    dtype = t.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float32 or t.get_device() != index or index < 0:
        raise ValueError(f"{name}: expected a tensor of bf16 or fp32 on cuda:{max(index, 0)}, got {t.device} {dtype}")
    return DT_FP32 if dtype is torch.float32 else DT_BF16


def launch_count():
    return int(library().trinity_sm100_launch_count())


def device_status(clear=False):
    value = ctypes.c_uint32(0)
    _check(library().trinity_sm100_device_status(ctypes.byref(value), int(clear)))
    return value.value


def gemm_pair_capacity():
    """CTA pairs the current device keeps resident at once in the GEMM's pair mode."""
    value = ctypes.c_int32(0)
    _check(library().trinity_sm100_gemm_pair_capacity(ctypes.byref(value)))
    return value.value


def set_wait_budget(cycles):
    """Budget of every bounded in-kernel wait on the current device, in SM clock cycles
    (0 restores the default of about two seconds)."""
    _check(library().trinity_sm100_set_wait_budget(int(cycles)))


def gemm(a, b, *, bias=None, bias_mode=None, activation=ACT_NONE, b2=None, out=None,
         out_dtype=torch.bfloat16, stream=None):
    """out = act(a @ b + bias); see ``trinity_sm100_gemm_bf16``.  Row-major 2-D tensors."""
    _require(a, torch.bfloat16, "a")
    _require(b, torch.bfloat16, "b")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError("gemm: a must be [m,k] and b [k,n]")
    if a.stride(1) != 1 or b.stride(1) != 1:
        raise ValueError("gemm: operands must be row-major with unit inner stride")
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if out.shape != (m, n) or out.stride(1) != 1:
        raise ValueError("gemm: out must be a row-major [m,n] tensor")
    args = GemmArgs()
    args.a, args.b, args.out = a.data_ptr(), b.data_ptr(), out.data_ptr()
    args.m, args.n, args.k = m, n, k
    args.lda, args.ldb, args.ldo = a.stride(0), b.stride(0), out.stride(0)
    args.activation = activation
    args.out_dtype = DT_FP32 if out.dtype == torch.float32 else DT_BF16
    if out.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("gemm: out dtype must be bf16 or fp32")
    if b2 is not None:
        _require(b2, torch.bfloat16, "b2")
        if b2.shape != b.shape or b2.stride() != b.stride():
            raise ValueError("gemm: b2 must match b")
        args.b2 = b2.data_ptr()
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
        if bias_mode is None:
            bias_mode = BIAS_MATRIX if bias.dim() == 2 else BIAS_COL_VECTOR
        expected = {BIAS_COL_VECTOR: (n,), BIAS_ROW_VECTOR: (m,), BIAS_MATRIX: (m, n)}[bias_mode]
        if tuple(bias.shape) != expected or bias.stride(-1) != 1:
            raise ValueError(f"gemm: bias shape {tuple(bias.shape)} does not fit mode {bias_mode}")
        args.bias = bias.data_ptr()
        args.ld_bias = bias.stride(0) if bias.dim() == 2 else 0
        args.bias_mode = bias_mode
    with torch.cuda.device(a.device):
        _check(library().trinity_sm100_gemm_bf16(ctypes.byref(args), _stream(stream)))
    return out


def gemm_batched(a, b, *, bias=None, activation=ACT_NONE, out=None, out_dtype=torch.bfloat16, stream=None):
    """out[z] = act(a[z] @ b[z] + bias[z]) for every batch entry z in one launch; see
    ``trinity_sm100_gemm_batched_bf16``.  ``a`` is [batch, m, k] and ``out`` [batch, m, n], any
    strides with a unit inner stride (so ``x.permute(1, 0, 2)`` of a [tokens, heads, k] tensor is
    fine); ``b`` is [batch, k, n] or a shared [k, n]; ``bias`` is [batch, n] or a shared [n]."""
    _require(a, torch.bfloat16, "a")
    _require(b, torch.bfloat16, "b")
    if a.dim() != 3 or b.dim() not in (2, 3) or a.shape[2] != b.shape[-2] or a.stride(2) != 1 or b.stride(-1) != 1:
        raise ValueError("gemm_batched: a must be [batch,m,k], b [batch,k,n] or [k,n], unit inner strides")
    batch, m, k = a.shape
    n = b.shape[-1]
    if b.dim() == 3 and b.shape[0] != batch:
        raise ValueError("gemm_batched: a and b disagree on the batch")
    if out is None:
        out = torch.empty((batch, m, n), dtype=out_dtype, device=a.device)
    if tuple(out.shape) != (batch, m, n) or out.stride(2) != 1 or out.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("gemm_batched: out must be [batch,m,n] with a unit inner stride, bf16 or fp32")
    args = GemmArgs()
    args.a, args.b, args.out = a.data_ptr(), b.data_ptr(), out.data_ptr()
    args.m, args.n, args.k = m, n, k
    args.lda, args.ldb, args.ldo = a.stride(1), b.stride(-2), out.stride(1)
    args.activation = activation
    args.out_dtype = DT_FP32 if out.dtype == torch.float32 else DT_BF16
    how = GemmBatchArgs()
    how.batch = batch
    how.stride_a, how.stride_out = a.stride(0), out.stride(0)
    how.stride_b = b.stride(0) if b.dim() == 3 else 0
    if bias is not None:
        _require(bias, torch.bfloat16, "bias")
        if tuple(bias.shape) not in ((n,), (batch, n)) or bias.stride(-1) != 1:
            raise ValueError("gemm_batched: bias must be [n] or [batch,n]")
        args.bias = bias.data_ptr()
        args.bias_mode = BIAS_COL_VECTOR
        how.stride_bias = bias.stride(0) if bias.dim() == 2 else 0
    with torch.cuda.device(a.device):
        _check(library().trinity_sm100_gemm_batched_bf16(ctypes.byref(args), ctypes.byref(how), _stream(stream)))
    return out


def gemm_adapters_workspace_bytes(m, n, rank):
    """Bytes of workspace that ``gemm_adapters`` needs."""
    return int(library().trinity_sm100_gemm_adapters_workspace_bytes(m, n, rank))


def gemm_adapters(x, w, down, up, index, *, scales=None, bias=None, activation=ACT_NONE, out=None,
                  out_dtype=torch.bfloat16, workspace=None, stream=None):
    """out[i] = act(x[i] @ w + bias + scales[z] * (x[i] @ down[z]) @ up[z]) with z = index[i] (negative: no
    adapter); see ``trinity_sm100_gemm_adapters_bf16``.

    ``x`` [m, k] and ``w`` [k, n] as in ``gemm``; ``down`` [adapters, k, rank] and ``up``
    [adapters, rank, n] BF16 with a unit inner stride, ``index`` int32 [m], ``scales`` FP32 [adapters],
    ``bias`` BF16 [n].  ``workspace`` (uint8, ``gemm_adapters_workspace_bytes``) is allocated per call
    unless given; calls that may overlap need one each."""
    device = x.device
    at = x.get_device()
    _operand(x, torch.bfloat16, at, "x")
    _operand(w, torch.bfloat16, at, "w")
    _operand(down, torch.bfloat16, at, "down")
    _operand(up, torch.bfloat16, at, "up")
    _operand(index, torch.int32, at, "index")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[0] or not _rows_ok(x) or not _rows_ok(w):
        raise ValueError("gemm_adapters: x must be [m,k] and w [k,n], row-major with unit inner strides")
    m, k = x.shape
    n = w.shape[1]
    count, rank = down.shape[0], down.shape[-1]
    down_strides, up_strides = down.stride(), up.stride()
    if (down.shape != (count, k, rank) or up.shape != (count, rank, n) or down_strides[-1] != 1
            or up_strides[-1] != 1):
        raise ValueError("gemm_adapters: down must be [adapters,k,rank] and up [adapters,rank,n], unit inner strides")
    if tuple(index.shape) != (m,) or not index.is_contiguous():
        raise ValueError("gemm_adapters: index must be [m]")
    if scales is not None:
        _operand(scales, torch.float32, at, "scales")
        if tuple(scales.shape) != (count,) or not scales.is_contiguous():
            raise ValueError("gemm_adapters: scales must be [adapters]")
    if bias is not None:
        _operand(bias, torch.bfloat16, at, "bias")
        if tuple(bias.shape) != (n,) or not bias.is_contiguous():
            raise ValueError("gemm_adapters: bias must be [n]")
    if out is not None:
        out_dtype = out.dtype
        if tuple(out.shape) != (m, n) or not _rows_ok(out) or out.get_device() != at:
            raise ValueError("gemm_adapters: out must be a row-major [m,n] tensor")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("gemm_adapters: out dtype must be bf16 or fp32")
    if workspace is not None:
        _workspace_operand(workspace, at, "gemm_adapters")

    def launch(handle):
        o = torch.empty((m, n), dtype=out_dtype, device=device) if out is None else out
        room = workspace
        if room is None:
            room = torch.empty(gemm_adapters_workspace_bytes(m, n, rank), dtype=torch.uint8, device=device)
        args = GemmArgs(x.data_ptr(), w.data_ptr(), None, bias.data_ptr() if bias is not None else None, o.data_ptr(),
                        m, n, k, _pitch(x), _pitch(w), _pitch(o), 0,
                        BIAS_NONE if bias is None else BIAS_COL_VECTOR, activation,
                        DT_FP32 if out_dtype == torch.float32 else DT_BF16, 0)
        adapters = AdaptersArgs(down.data_ptr(), up.data_ptr(), index.data_ptr(),
                                scales.data_ptr() if scales is not None else None, room.data_ptr(),
                                room.numel() * room.element_size(), down_strides[1], down_strides[0],
                                up_strides[1], up_strides[0], count, rank)
        _check(library().trinity_sm100_gemm_adapters_bf16(ctypes.byref(args), ctypes.byref(adapters), handle))
        return o

    return _submit(device, stream, (x, w, down, up, index, scales, bias, out, workspace), launch)


def rmsnorm(x, gain=None, eps=0.0, out=None, stream=None):
    _require(x, torch.bfloat16, "x")
    if x.dim() != 2 or not x.is_contiguous():
        raise ValueError("rmsnorm: x must be a contiguous [rows, cols] tensor")
    if out is None:
        out = torch.empty_like(x)
    if gain is not None:
        _require(gain, torch.bfloat16, "gain")
        if tuple(gain.shape) != (x.shape[1],) or not gain.is_contiguous():
            raise ValueError("rmsnorm: gain must be [cols]")
    with torch.cuda.device(x.device):
        _check(library().trinity_sm100_rmsnorm_bf16(
            x.data_ptr(), gain.data_ptr() if gain is not None else None, out.data_ptr(),
            x.shape[0], x.shape[1], float(eps), _stream(stream)))
    return out


def _gain_operand(t, cols, index, name):
    _operand(t, torch.bfloat16, index, name)
    if t.shape != (cols,) or not t.is_contiguous():
        raise ValueError(f"rmsnorm_residual: {name} must be [cols]")


def _rows_operand(t, dtype, shape, index, name):
    _operand(t, dtype, index, name)
    if t.shape != shape or not _rows_ok(t):
        raise ValueError(f"rmsnorm_residual: {name} must be [rows, cols] with a unit inner stride")


def rmsnorm_residual(x, residual, *, gain=None, post_gain=None, post_norm=None, gate=None, residual_scale=1.0,
                     eps=0.0, post_eps=None, residual_out=None, out=None, stream=None):
    """The seam between two blocks: ``(h, y)`` with ``h = residual_scale * residual + gate * b`` and
    ``y = h / sqrt(mean(h^2) + eps) * gain``, where ``b`` is the block's output ``x``, normalised
    with ``post_eps`` (default ``eps``) and ``post_gain`` if ``post_norm`` (default: if ``post_gain``
    is given).  See ``trinity_sm100_rmsnorm_residual``.

    ``x`` and ``residual`` are [rows, cols], BF16 or FP32, with a unit inner stride; ``h`` has the
    residual's type, ``y`` is BF16.  ``gate`` is a BF16 tensor that broadcasts to [rows, cols]:
    [cols], [1, cols], [rows, 1] or [rows, cols].  ``residual_out=residual`` updates the stream in place."""
    device = x.device
    index = x.get_device()
    x_dtype = _real_operand(x, index, "x")
    residual_dtype = _real_operand(residual, index, "residual")
    shape = x.shape
    if residual.shape != shape or not _rows_ok(x) or not _rows_ok(residual):
        raise ValueError("rmsnorm_residual: x and residual must be [rows, cols] with a unit inner stride")
    rows, cols = shape
    if gain is not None:
        _gain_operand(gain, cols, index, "gain")
    if post_gain is not None:
        _gain_operand(post_gain, cols, index, "post_gain")
    if post_norm is None:
        post_norm = post_gain is not None
    elif not post_norm and post_gain is not None:
        raise ValueError("rmsnorm_residual: post_gain without the post norm")
    gate_pointer, row_stride, col_stride = None, 0, 0
    if gate is not None:
        _operand(gate, torch.bfloat16, index, "gate")
        if gate.shape != shape:
            try:
                gate = gate.expand(rows, cols)
            except RuntimeError:
                raise ValueError(f"rmsnorm_residual: gate {tuple(gate.shape)} does not broadcast to {(rows, cols)}") from None
        row_stride, col_stride = gate.stride()
        if cols == 1:
            col_stride = 0
        if rows == 1:
            row_stride = 0
        if col_stride not in (0, 1):
            raise ValueError("rmsnorm_residual: gate must have an inner stride of 0 or 1")
        gate_pointer = gate.data_ptr()
    if residual_out is not None:
        _rows_operand(residual_out, residual.dtype, shape, index, "residual_out")
    if out is not None:
        _rows_operand(out, torch.bfloat16, shape, index, "out")

    def launch(handle):
        if residual_out is None:
            h, h_pitch = _empty_rows(residual, residual.dtype), cols
        else:
            h, h_pitch = residual_out, _pitch(residual_out)
        if out is None:
            y, y_pitch = _empty_rows(x, torch.bfloat16), cols
        else:
            y, y_pitch = out, _pitch(out)
        args = RmsnormResidualArgs(
            x.data_ptr(), residual.data_ptr(), gate_pointer, None if gain is None else gain.data_ptr(),
            None if post_gain is None else post_gain.data_ptr(), h.data_ptr(), y.data_ptr(), rows, cols,
            _pitch(x), _pitch(residual), h_pitch, y_pitch, row_stride, col_stride, x_dtype, residual_dtype,
            bool(post_norm), eps, eps if post_eps is None else post_eps, residual_scale)
        _check(library().trinity_sm100_rmsnorm_residual(ctypes.byref(args), handle))
        return h, y

    return _submit(device, stream, (x, residual, gain, post_gain, gate, residual_out, out), launch)


def softmax(x, out=None, stream=None):
    _require(x, torch.bfloat16, "x")
    if x.dim() != 2 or not x.is_contiguous():
        raise ValueError("softmax: x must be a contiguous [rows, cols] tensor")
    if out is None:
        out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _check(library().trinity_sm100_softmax_bf16(
            x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], _stream(stream)))
    return out


def mla_default_splits(batch, seq):
    return int(library().trinity_sm100_mla_default_splits(batch, seq))


def mla_balanced_slots(batch, seq):
    return int(library().trinity_sm100_mla_balanced_slots(batch, seq))


def mla_scratch_bytes(batch, heads, d_v, kv_splits):
    return int(library().trinity_sm100_mla_scratch_bytes(batch, heads, d_v, kv_splits))


def mla_decode(q, cache, scale, d_v=512, kv_splits=0, out=None, scratch=None, stream=None):
    """out[b,h,:] = softmax_s(scale * q[b,h] . cache[b,s]) @ cache[b,:,:d_v]."""
    _require(q, torch.bfloat16, "q")
    _require(cache, torch.bfloat16, "cache")
    if q.dim() != 3 or cache.dim() != 3 or not q.is_contiguous() or not cache.is_contiguous():
        raise ValueError("mla_decode: q [batch,heads,d_qk] and cache [batch,seq,d_qk], contiguous")
    batch, heads, d_qk = q.shape
    if cache.shape[0] != batch or cache.shape[2] != d_qk:
        raise ValueError("mla_decode: q and cache disagree on batch or width")
    seq = cache.shape[1]
    if out is None:
        out = torch.empty((batch, heads, d_v), dtype=torch.bfloat16, device=q.device)
    # kv_splits == 0 leaves the schedule to the library, kv_splits < 0 asks for the balanced one;
    # either way the library says how many partial slots per sequence it needs scratch for.
    slots = kv_splits if kv_splits > 0 else (
        mla_default_splits(batch, seq) if kv_splits == 0 else mla_balanced_slots(batch, seq))
    need = mla_scratch_bytes(batch, heads, d_v, slots)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    args = MlaArgs()
    args.q, args.cache, args.out = q.data_ptr(), cache.data_ptr(), out.data_ptr()
    args.scratch, args.scratch_bytes = scratch.data_ptr(), scratch.numel() * scratch.element_size()
    args.batch, args.heads, args.seq, args.d_qk, args.d_v = batch, heads, seq, d_qk, d_v
    args.kv_splits = kv_splits
    args.scale = float(scale)
    with torch.cuda.device(q.device):
        _check(library().trinity_sm100_mla_decode_bf16(ctypes.byref(args), _stream(stream)))
    return out


MLA_STATIC_SCRATCH_BYTES = 32 << 20


def mla_decode_noalloc(q, cache, scale, d_v=512, kv_splits=0, out=None, stream=None):
    """``mla_decode`` for callers that cannot bring or allocate scratch memory: the split
    partials live in a fixed array inside the kernel library (``MLA_STATIC_SCRATCH_BYTES`` per
    GPU).  ``out`` must be passed by such callers; it is created here only as a convenience for
    tests.  Calls that overlap on one GPU race on the shared array."""
    _require(q, torch.bfloat16, "q")
    _require(cache, torch.bfloat16, "cache")
    if q.dim() != 3 or cache.dim() != 3 or not q.is_contiguous() or not cache.is_contiguous():
        raise ValueError("mla_decode: q [batch,heads,d_qk] and cache [batch,seq,d_qk], contiguous")
    batch, heads, d_qk = q.shape
    if cache.shape[0] != batch or cache.shape[2] != d_qk:
        raise ValueError("mla_decode: q and cache disagree on batch or width")
    if out is None:
        out = torch.empty((batch, heads, d_v), dtype=torch.bfloat16, device=q.device)
    args = MlaArgs()
    args.q, args.cache, args.out = q.data_ptr(), cache.data_ptr(), out.data_ptr()
    args.batch, args.heads, args.seq, args.d_qk, args.d_v = batch, heads, cache.shape[1], d_qk, d_v
    args.kv_splits = kv_splits
    args.scale = float(scale)
    with torch.cuda.device(q.device):
        _check(library().trinity_sm100_mla_decode_bf16_noalloc(ctypes.byref(args), _stream(stream)))
    return out


class Kv4Cache:
    """A paged key/value cache held in 4 bits (see ``trinity_sm100_kv4_cache`` for the format):
    codes uint8 [pages, kv_heads, page, head_dim / 2], scales BF16 [pages, kv_heads, page,
    head_dim / group, 2] with (scale, zero) pairs.  ``kv4_cache`` makes an empty one."""

    def __init__(self, k_codes, k_scales, v_codes, v_scales):
        codes, scales = k_codes.shape, k_scales.shape
        if len(codes) != 4 or len(scales) != 5 or scales[4] != 2:
            raise ValueError("Kv4Cache: codes are [pages, kv_heads, page, head_dim / 2], "
                             "scales [pages, kv_heads, page, head_dim / group, 2]")
        pages, kv_heads, page, half = codes
        groups = scales[3]
        if (scales[:3] != codes[:3] or v_codes.shape != codes or v_scales.shape != scales
                or groups == 0 or (2 * half) % groups):
            raise ValueError("Kv4Cache: codes and scales disagree")
        index = k_codes.get_device()
        _operand(k_codes, torch.uint8, index, "k_codes")
        _operand(v_codes, torch.uint8, index, "v_codes")
        _operand(k_scales, torch.bfloat16, index, "k_scales")
        _operand(v_scales, torch.bfloat16, index, "v_scales")
        if not (k_codes.is_contiguous() and v_codes.is_contiguous() and k_scales.is_contiguous()
                and v_scales.is_contiguous()):
            raise ValueError("Kv4Cache: the tensors must be contiguous")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.pages, self.kv_heads, self.page = pages, kv_heads, page
        self.head_dim, self.group = 2 * half, 2 * half // groups
        self.device, self.index = k_codes.device, index
        self.args = Kv4CacheArgs(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                                 pages, kv_heads, page, self.head_dim, self.group, 0)

    @property
    def tensors(self):
        return self.k_codes, self.k_scales, self.v_codes, self.v_scales


def kv4_cache(pages, kv_heads, page, head_dim, group=None, device="cuda"):
    """An empty ``Kv4Cache`` of ``pages`` pages of ``page`` positions, quantised in groups of
    ``group`` channels (default: the whole head)."""
    group = head_dim if group is None else group
    if group <= 0 or head_dim % group:
        raise ValueError(f"kv4_cache: groups of {group} do not divide {head_dim} channels")
    codes = [torch.zeros((pages, kv_heads, page, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.zeros((pages, kv_heads, page, head_dim // group, 2), dtype=torch.bfloat16, device=device)
              for _ in range(2)]
    return Kv4Cache(codes[0], scales[0], codes[1], scales[1])


def _kv4_rows(what, cache, k, v, slots):
    tokens = slots.shape[0] if slots.dim() == 1 else -1
    expected = (tokens, cache.kv_heads, cache.head_dim)
    ks, vs = k.stride(), v.stride()
    if k.shape != expected or v.shape != expected or ks[2] != 1 or vs[2] != 1:
        raise ValueError(f"{what}: k and v must be [tokens, {cache.kv_heads}, {cache.head_dim}] with a unit inner "
                         "stride and slots [tokens]")
    _operand(slots, torch.int64, cache.index, "slots")
    if not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be contiguous")
    return Kv4RowsArgs(k.data_ptr(), v.data_ptr(), slots.data_ptr(), tokens, ks[0], ks[1], vs[0], vs[1])


def kv4_append(cache, k, v, slots, stream=None):
    """Quantises the BF16 rows ``k`` and ``v`` [tokens, kv_heads, head_dim] (views with any token and
    head stride) into ``cache`` at positions ``slots`` (int64 [tokens]; distinct; negative: token not
    written); see ``trinity_sm100_kv4_append``."""
    _operand(k, torch.bfloat16, cache.index, "k")
    _operand(v, torch.bfloat16, cache.index, "v")
    args = _kv4_rows("kv4_append", cache, k, v, slots)

    def launch(handle):
        _check(library().trinity_sm100_kv4_append(ctypes.byref(cache.args), ctypes.byref(args), handle))

    _submit(cache.device, stream, (k, v, slots, *cache.tensors), launch)


def kv4_read(cache, slots, *, dtype=torch.bfloat16, k_out=None, v_out=None, stream=None):
    """The keys and values [tokens, kv_heads, head_dim] that ``cache`` holds at positions ``slots``
    (int64 [tokens]; negative: zeros), in BF16 or FP32; see ``trinity_sm100_kv4_read``."""
    if (k_out is None) != (v_out is None):
        raise ValueError("kv4_read: give both outputs or none")
    if k_out is not None:
        dtype = k_out.dtype
        _operand(k_out, dtype, cache.index, "k_out")
        _operand(v_out, dtype, cache.index, "v_out")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("kv4_read: dtype must be bf16 or fp32")
    code = DT_FP32 if dtype == torch.float32 else DT_BF16

    def launch(handle):
        if k_out is None:
            shape = (slots.shape[0] if slots.dim() == 1 else -1, cache.kv_heads, cache.head_dim)
            if shape[0] < 0:
                raise ValueError("kv4_read: slots must be [tokens]")
            k = torch.empty(shape, dtype=dtype, device=cache.device)
            v = torch.empty_like(k)
        else:
            k, v = k_out, v_out
        args = _kv4_rows("kv4_read", cache, k, v, slots)
        _check(library().trinity_sm100_kv4_read(ctypes.byref(cache.args), ctypes.byref(args), code, handle))
        return k, v

    return _submit(cache.device, stream, (slots, k_out, v_out, *cache.tensors), launch)


_kv4_workspaces = {}


def kv4_decode_workspace_bytes(heads, kv_heads, head_dim):
    """Bytes of workspace that ``kv4_decode`` needs on the current device."""
    key = (torch._C._cuda_getDevice(), heads, kv_heads, head_dim)
    size = _kv4_workspaces.get(key)
    if size is None:
        size = int(library().trinity_sm100_kv4_decode_workspace_bytes(heads, kv_heads, head_dim))
        if size:      # 0: no such layout, or the device could not be asked
            _kv4_workspaces[key] = size
    return size


def kv4_decode(q, cache, page_table, lengths, scale, *, out=None, lse=None, workspace=None, stream=None):
    """Attention of one new token per sequence over a 4-bit paged cache: ``out[b, h] =
    softmax_t(scale * q[b, h] . k[b, t]) v[b, t]`` over the first ``lengths[b]`` positions, which lie in
    the pages ``page_table[b]``; see ``trinity_sm100_kv4_decode``.

    ``q`` is BF16 [batch, heads, head_dim] (views allowed), ``page_table`` int32 [batch, max_pages],
    ``lengths`` int32 [batch] on the device.  ``lse`` (FP32 [batch, heads]) receives the logarithm of
    the sum of exponentials.  ``workspace`` (uint8, ``kv4_decode_workspace_bytes``) is allocated per
    call unless given; calls that may overlap need one each."""
    device, index = cache.device, cache.index
    _operand(q, torch.bfloat16, index, "q")
    _operand(page_table, torch.int32, index, "page_table")
    _operand(lengths, torch.int32, index, "lengths")
    if q.dim() != 3 or q.shape[2] != cache.head_dim or q.stride(2) != 1:
        raise ValueError(f"kv4_decode: q must be [batch, heads, {cache.head_dim}] with a unit inner stride")
    batch, heads, head_dim = q.shape
    if (not _rows_ok(page_table) or page_table.shape[0] != batch or lengths.shape != (batch,)
            or not lengths.is_contiguous()):
        raise ValueError("kv4_decode: page_table must be [batch, max_pages] and lengths [batch]")
    if out is not None:
        _operand(out, torch.bfloat16, index, "out")
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError("kv4_decode: out must be a contiguous [batch, heads, head_dim] tensor")
    if lse is not None:
        _operand(lse, torch.float32, index, "lse")
        if lse.shape != (batch, heads) or not lse.is_contiguous():
            raise ValueError("kv4_decode: lse must be a contiguous [batch, heads] tensor")
    if workspace is not None:
        _workspace_operand(workspace, index, "kv4_decode")

    def launch(handle):
        o = _empty_rows(q, torch.bfloat16) if out is None else out
        room = workspace
        if room is None:
            room = torch.empty(kv4_decode_workspace_bytes(heads, cache.kv_heads, head_dim), dtype=torch.uint8,
                               device=device)
        args = Kv4DecodeArgs(q.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), o.data_ptr(),
                             lse.data_ptr() if lse is not None else None, room.data_ptr(),
                             room.numel() * room.element_size(), q.stride(0), q.stride(1),
                             _pitch(page_table), batch, heads, page_table.shape[1], scale)
        _check(library().trinity_sm100_kv4_decode(ctypes.byref(cache.args), ctypes.byref(args), handle))
        return o

    return _submit(device, stream, (q, page_table, lengths, out, lse, workspace, *cache.tensors), launch)


def allreduce_flag_words():
    return int(library().trinity_sm100_allreduce_flag_words())


def allreduce(peer_ptrs, flag_ptrs, rows, cols, rank, epoch, stream=None):
    """In-place sum all-reduce over peer-mapped BF16 buffers (see the C header)."""
    world = len(peer_ptrs)
    peers = (ctypes.c_void_p * world)(*peer_ptrs)
    flags = (ctypes.c_void_p * world)(*flag_ptrs)
    args = AllReduceArgs()
    args.peers = ctypes.cast(peers, ctypes.POINTER(ctypes.c_void_p))
    args.flags = ctypes.cast(flags, ctypes.POINTER(ctypes.c_void_p))
    args.rows, args.cols, args.world, args.rank, args.epoch = rows, cols, world, rank, epoch
    _check(library().trinity_sm100_allreduce_bf16(ctypes.byref(args), _stream(stream)))


PEER_TABLE_BYTES = 1024
PEER_BUFFERS = 4


def peer_table(world, rank, workspace_ptrs, buffer_ptrs):
    """The bytes of a ``trinity_sm100_peer_table`` (see the C header): ``workspace_ptrs[r]`` is
    rank r's workspace as mapped into this process, ``buffer_ptrs[i][r]`` rank r's copy of the
    i-th symmetric plan buffer."""
    import struct
    if len(buffer_ptrs) > PEER_BUFFERS or world > 8:
        raise ValueError("at most %d symmetric buffers and 8 ranks" % PEER_BUFFERS)
    words = struct.pack("<iiIIIIII", world, rank, 0, 0, 0, 0, 0, 0)
    words += struct.pack("<8Q", *(list(workspace_ptrs) + [0] * (8 - world)))
    for i in range(PEER_BUFFERS):
        ptrs = list(buffer_ptrs[i]) if i < len(buffer_ptrs) else []
        words += struct.pack("<8Q", *(ptrs + [0] * (8 - len(ptrs))))
    words += bytes(64 * 4)
    return words + bytes(PEER_TABLE_BYTES - len(words))


def allgather(workspace_ptr, source, out, rows, cols, axis, world, stream=None):
    """out = rank-major all-gather of the [rows, cols] BF16 shards held in symmetric buffer
    ``source`` of the peer table at ``workspace_ptr`` (see ``trinity_sm100_allgather_bf16``)."""
    _require(out, torch.bfloat16, "out")
    with torch.cuda.device(out.device):
        _check(library().trinity_sm100_allgather_bf16(ctypes.c_void_p(workspace_ptr), source, out.data_ptr(),
                                                      rows, cols, axis, world, _stream(stream)))
    return out


def gemm_allreduce_stamps():
    """Milestones (ns of the device timer) of the most recent fused launch's first thread block:
    start, last MMA committed, last partial tile handed over, last owned rows reduced, retired."""
    values = (ctypes.c_uint64 * 5)()
    _check(library().trinity_sm100_gemm_allreduce_stamps(values))
    return list(values)


def gemm_allreduce_flag_words(m, n, world):
    return int(library().trinity_sm100_gemm_allreduce_flag_words(m, n, world))


def gemm_allreduce(a, b, out, peer_ptrs, flag_ptrs, rank, epoch, stream=None):
    """out (on every rank) = sum over ranks of a_rank @ b_rank, reduced inside the GEMM's
    epilogue over peer-mapped memory (see ``trinity_sm100_gemm_allreduce_bf16``).  ``out`` is this
    rank's symmetric buffer, ``peer_ptrs[rank] == out.data_ptr()``."""
    _require(a, torch.bfloat16, "a")
    _require(b, torch.bfloat16, "b")
    _require(out, torch.bfloat16, "out")
    m, kk = a.shape
    n = b.shape[1]
    args = GemmArgs()
    args.a, args.b, args.out = a.data_ptr(), b.data_ptr(), out.data_ptr()
    args.m, args.n, args.k = m, n, kk
    args.lda, args.ldb, args.ldo = a.stride(0), b.stride(0), out.stride(0)
    world = len(peer_ptrs)
    peers = (ctypes.c_void_p * world)(*peer_ptrs)
    flags = (ctypes.c_void_p * world)(*flag_ptrs)
    red = AllReduceArgs()
    red.peers = ctypes.cast(peers, ctypes.POINTER(ctypes.c_void_p))
    red.flags = ctypes.cast(flags, ctypes.POINTER(ctypes.c_void_p))
    red.rows, red.cols, red.world, red.rank, red.epoch = m, n, world, rank, epoch
    with torch.cuda.device(a.device):
        _check(library().trinity_sm100_gemm_allreduce_bf16(ctypes.byref(args), ctypes.byref(red),
                                                           _stream(stream)))
    return out
