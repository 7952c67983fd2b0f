"""ctypes binding of the C ABI in ``include/quant_ops_hip.h``.

This is the FFI view of ``libquant_ops_hip.so``: plain device pointers, sizes,
strides and a stream handle, no torch types. Tests and the benchmark call the
kernels through it; torch tensors are only used here to own device memory and
to name the current stream. Every call raises ``QuantOpsError`` on a non-zero
status, with the library's message.
"""
import contextlib
import ctypes
import os

import torch

from ._loader import HIP_LIB_PATH

DTYPE_F32, DTYPE_F16, DTYPE_BF16, DTYPE_I8, DTYPE_I32 = 0, 1, 2, 3, 4
MX_FP4, MX_FP8 = 0, 1
STATUS = {0: "QO_OK", 1: "QO_ERR_NULL_POINTER", 2: "QO_ERR_SHAPE", 3: "QO_ERR_DTYPE",
          4: "QO_ERR_ALIGNMENT", 5: "QO_ERR_UNSUPPORTED", 6: "QO_ERR_LAUNCH"}

# Every symbol the header declares; the CPU tests check they are all exported.
EXPORTED = ("qo_status_string", "qo_version", "qo_last_error", "qo_set_kernel_routing", "qo_flatquant_quantize",
            "qo_int4_gemm", "qo_int4_gemm_bias", "qo_int4_gemm_ws", "qo_int4_gemm_workspace_size", "qo_int4_gemm_workspace_needed", "qo_int4_gemm_f6_workspace_bytes",
            "qo_int4_gemm_f6_prepare", "qo_int4_gemm_f6_run", "qo_int4_gemm_f6_operand_bytes",
            "qo_int4_gemm_f6_convert", "qo_int4_gemm_f6_run2", "qo_w4a4_linear_f6w", "qo_w4a4_linear", "qo_w4a4_linear_ws", "qo_w4a4_linear_noalloc", "qo_dequantize_int4",
            "qo_pack_int4_to_int32", "qo_pack_int4_clamped", "qo_unpack_int32_to_int4", "qo_transpose_int32",
            "qo_mx_quantize", "qo_mx_dequantize", "qo_rms_norm_mx_quantize", "qo_swiglu_mx_quantize", "qo_mx_gemm",
            "qo_mx_gemm_workspace_size", "qo_kv4_append", "qo_kv4_read", "qo_kv4_attention",
            "qo_kv4_attention_workspace_size")

# QO_ROUTE_* bits of qo_set_kernel_routing (include/quant_ops_hip.h)
ROUTE = {"FQ_GENERIC": 1 << 0, "FQ_NO_WAVE": 1 << 1, "FQ_NO_DUO": 1 << 2, "FQ_NO_FEW": 1 << 3,
         "GEMM_GENERIC": 1 << 4, "GEMM_NO_DMA": 1 << 5, "GEMM_NO_SKINNY": 1 << 6,
         "LINEAR_NO_READ_AHEAD": 1 << 7, "GEMM_NO_F6": 1 << 8}

_TORCH_CODE = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


class KV4Struct(ctypes.Structure):
    """``qo_kv4_cache``."""

    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p), ("params", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32)]


class HeadsStruct(ctypes.Structure):
    """``qo_heads``."""

    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class QuantOpsError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"{STATUS.get(status, status)}: {message}")
        self.status = status


_lib = None


def lib():
    """Load (once) and return the ctypes handle with argument types set."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(HIP_LIB_PATH):
        raise QuantOpsError(5, f"{HIP_LIB_PATH} is not built")
    L = ctypes.CDLL(HIP_LIB_PATH)
    c_i64, c_int, c_vp, c_f = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_float
    L.qo_status_string.restype = ctypes.c_char_p
    L.qo_status_string.argtypes = [c_int]
    L.qo_version.restype = ctypes.c_char_p
    L.qo_version.argtypes = []
    L.qo_last_error.restype = ctypes.c_char_p
    L.qo_last_error.argtypes = []
    L.qo_set_kernel_routing.restype = ctypes.c_uint
    L.qo_set_kernel_routing.argtypes = [ctypes.c_uint]
    L.qo_flatquant_quantize.restype = c_int
    L.qo_flatquant_quantize.argtypes = [c_vp, c_int, c_i64, c_i64, c_vp, c_vp, c_int, c_int, c_f, c_int,
                                        c_vp, c_vp, c_vp]
    L.qo_int4_gemm.restype = c_int
    L.qo_int4_gemm.argtypes = [c_vp, c_i64, c_vp, c_i64, c_i64, c_vp, c_int, c_vp, c_int, c_vp, c_int, c_i64,
                               c_i64, c_i64, c_i64, c_vp]
    L.qo_int4_gemm_bias.restype = c_int
    L.qo_int4_gemm_bias.argtypes = [c_vp, c_i64, c_vp, c_i64, c_i64, c_vp, c_int, c_vp, c_int, c_vp, c_vp, c_int,
                                    c_i64, c_i64, c_i64, c_i64, c_vp]
    L.qo_int4_gemm_ws.restype = c_int
    L.qo_int4_gemm_ws.argtypes = [c_vp, c_i64, c_vp, c_i64, c_i64, c_vp, c_int, c_vp, c_int, c_vp, c_vp, c_int,
                                  c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp]
    L.qo_int4_gemm_workspace_size.restype = c_i64
    L.qo_int4_gemm_workspace_size.argtypes = [c_i64, c_i64, c_i64, c_int]
    L.qo_int4_gemm_workspace_needed.restype = c_i64
    L.qo_int4_gemm_workspace_needed.argtypes = [c_vp, c_i64, c_vp, c_i64, c_i64, c_vp, c_int, c_i64, c_i64, c_i64, c_i64]
    L.qo_int4_gemm_f6_workspace_bytes.restype = c_i64
    L.qo_int4_gemm_f6_workspace_bytes.argtypes = [c_i64, c_i64, c_i64]
    L.qo_int4_gemm_f6_prepare.restype = c_int
    L.qo_int4_gemm_f6_prepare.argtypes = [c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp]
    L.qo_int4_gemm_f6_run.restype = c_int
    L.qo_int4_gemm_f6_run.argtypes = [c_vp, c_int, c_vp, c_int, c_vp, c_vp, c_int, c_i64, c_i64, c_i64, c_i64, c_vp,
                                      c_i64, c_vp]
    L.qo_w4a4_linear.restype = c_int
    L.qo_w4a4_linear.argtypes = [c_vp, c_int, c_i64, c_i64, c_vp, c_vp, c_int, c_int, c_f, c_vp, c_i64, c_i64,
                                 c_vp, c_int, c_vp, c_vp, c_vp, c_vp, c_i64, c_vp]
    L.qo_w4a4_linear_ws.restype = c_int
    L.qo_w4a4_linear_ws.argtypes = [c_vp, c_int, c_i64, c_i64, c_vp, c_vp, c_int, c_int, c_f, c_vp, c_i64, c_i64,
                                    c_vp, c_int, c_vp, c_vp, c_vp, c_vp, c_i64, c_vp, c_i64, c_vp]
    L.qo_int4_gemm_f6_operand_bytes.restype = c_i64
    L.qo_int4_gemm_f6_operand_bytes.argtypes = [c_i64, c_i64]
    L.qo_int4_gemm_f6_convert.restype = c_int
    L.qo_int4_gemm_f6_convert.argtypes = [c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp]
    L.qo_int4_gemm_f6_run2.restype = c_int
    L.qo_int4_gemm_f6_run2.argtypes = [c_vp, c_i64, c_vp, c_i64, c_vp, c_int, c_vp, c_int, c_vp, c_vp, c_int, c_i64,
                                       c_i64, c_i64, c_i64, c_vp]
    L.qo_w4a4_linear_f6w.restype = c_int
    L.qo_w4a4_linear_f6w.argtypes = [c_vp, c_int, c_i64, c_i64, c_vp, c_vp, c_int, c_int, c_f, c_vp, c_i64, c_i64,
                                     c_vp, c_int, c_vp, c_vp, c_vp, c_vp, c_i64, c_vp, c_i64, c_vp]
    L.qo_w4a4_linear_noalloc.restype = c_int
    L.qo_w4a4_linear_noalloc.argtypes = [c_vp, c_int, c_i64, c_i64, c_vp, c_vp, c_int, c_int, c_f, c_vp, c_i64,
                                         c_i64, c_vp, c_int, c_vp, c_vp, c_i64, c_vp]
    L.qo_dequantize_int4.restype = c_int
    L.qo_dequantize_int4.argtypes = [c_vp, c_int, c_vp, c_int, c_i64, c_i64, c_vp, c_vp]
    for name in ("qo_pack_int4_to_int32", "qo_pack_int4_clamped", "qo_unpack_int32_to_int4", "qo_transpose_int32"):
        fn = getattr(L, name)
        fn.restype = c_int
        fn.argtypes = [c_vp, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp]
    L.qo_mx_quantize.restype = c_int
    L.qo_mx_quantize.argtypes = [c_vp, c_int, c_i64, c_i64, c_i64, c_int, c_vp, c_vp, c_i64, c_vp]
    L.qo_mx_dequantize.restype = c_int
    L.qo_mx_dequantize.argtypes = [c_vp, c_vp, c_i64, c_int, c_i64, c_i64, c_vp, c_int, c_vp]
    L.qo_rms_norm_mx_quantize.restype = c_int
    L.qo_rms_norm_mx_quantize.argtypes = [c_vp, c_vp, c_int, c_i64, c_i64, c_i64, c_i64, c_vp, c_int, c_f, c_int,
                                          c_vp, c_vp, c_i64, c_vp, c_vp]
    L.qo_swiglu_mx_quantize.restype = c_int
    L.qo_swiglu_mx_quantize.argtypes = [c_vp, c_int, c_i64, c_i64, c_i64, c_int, c_vp, c_vp, c_i64, c_vp]
    L.qo_mx_gemm.restype = c_int
    L.qo_mx_gemm.argtypes = [c_vp, c_i64, c_int, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_int, c_i64,
                             c_i64, c_i64, c_i64, c_vp, c_i64, c_vp]
    L.qo_mx_gemm_workspace_size.restype = c_i64
    L.qo_mx_gemm_workspace_size.argtypes = [c_i64, c_i64, c_i64, c_int]
    c_cache, c_heads = ctypes.POINTER(KV4Struct), ctypes.POINTER(HeadsStruct)
    L.qo_kv4_append.restype = c_int
    L.qo_kv4_append.argtypes = [c_cache, c_heads, c_heads, c_heads, c_int, c_i64, c_int, c_vp, c_vp, c_vp, c_vp, c_i64, c_int,
                                c_int, c_vp, c_vp]
    L.qo_kv4_read.restype = c_int
    L.qo_kv4_read.argtypes = [c_cache, c_vp, c_i64, c_vp, c_vp, c_int, c_vp]
    L.qo_kv4_attention.restype = c_int
    L.qo_kv4_attention.argtypes = [c_cache, c_heads, c_int, c_i64, c_int, c_vp, c_i64, c_i64, c_vp, c_vp, c_i64, c_f, c_i64,
                                   c_vp, c_vp, c_i64, c_vp]
    L.qo_kv4_attention_workspace_size.restype = c_i64
    L.qo_kv4_attention_workspace_size.argtypes = [c_cache, c_int, c_i64, c_int, c_i64, c_i64, c_int, c_i64]
    _lib = L
    return L


def _check(status):
    if status != 0:
        raise QuantOpsError(status, lib().qo_last_error().decode())


def _stream(stream):
    if stream is None:
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    if isinstance(stream, torch.cuda.Stream):
        return ctypes.c_void_p(stream.cuda_stream)
    return ctypes.c_void_p(stream)


def version() -> str:
    return lib().qo_version().decode()


def set_kernel_routing(mask: int) -> int:
    """Set the process-wide QO_ROUTE_* mask; returns the previous one."""
    return int(lib().qo_set_kernel_routing(mask))


def route_mask(*names) -> int:
    mask = 0
    for name in names:
        mask |= ROUTE[name]
    return mask


@contextlib.contextmanager
def kernel_routing(*names):
    """Add the named QO_ROUTE_* bits (``ROUTE`` keys) for the duration of the block."""
    prev = set_kernel_routing(0)
    set_kernel_routing(prev | route_mask(*names))
    try:
        yield
    finally:
        set_kernel_routing(prev)


def flatquant_quantize(x, left, right, clip_ratio=1.0, pack_int32=False, out_codes=None, out_scales=None,
                       stream=None):
    """Call ``qo_flatquant_quantize`` on device tensors; allocates outputs if not given.

    The C ABI reads L and R as row-major [M, M] / [N, N]; other layouts (e.g. the
    column-major Q that torch.linalg.qr returns) are made contiguous here.
    """
    t, f = x.shape
    if x.stride(1) != 1:
        x = x.contiguous()
    left, right = left.contiguous(), right.contiguous()
    m, n = left.shape[0], right.shape[0]
    if out_codes is None:
        out_codes = torch.empty((t, f // 8) if pack_int32 else (t, f),
                                dtype=torch.int32 if pack_int32 else torch.int8, device=x.device)
    if out_scales is None:
        out_scales = torch.empty((t,), dtype=torch.float32, device=x.device)
    _check(lib().qo_flatquant_quantize(
        ctypes.c_void_p(x.data_ptr()), _TORCH_CODE[x.dtype], t, x.stride(0) if t else f,
        ctypes.c_void_p(left.data_ptr()), ctypes.c_void_p(right.data_ptr()), m, n,
        float(clip_ratio), 1 if pack_int32 else 0,
        ctypes.c_void_p(out_codes.data_ptr()), ctypes.c_void_p(out_scales.data_ptr()), _stream(stream)))
    return out_codes, out_scales


def gemm_workspace_size(m, n, k, out_dtype=torch.float16):
    """``qo_int4_gemm_workspace_size``: bytes of the FP6 route's workspace, whatever the operands' layout
    (0: not taken)."""
    return int(lib().qo_int4_gemm_workspace_size(m, n, k, _TORCH_CODE[out_dtype]))


def int4_gemm(a, b, scale_a, scale_b, out_dtype=torch.float16, out=None, stream=None, bias=None,
              workspace=None):
    """Call ``qo_int4_gemm`` (``qo_int4_gemm_bias`` with ``bias``, converted to the
    output dtype); ``b`` may be row-major [K/8, N] or the ``W.t()`` view. With
    ``workspace`` (a uint8 device tensor, or True to allocate one of
    gemm_workspace_size bytes) the call goes to ``qo_int4_gemm_ws``."""
    m, kp = a.shape
    if a.stride(1) != 1:
        a = a.contiguous()
    if b.stride(0) != 1 and b.stride(1) != 1:
        b = b.contiguous()
    scale_a, scale_b = scale_a.contiguous(), scale_b.contiguous()
    n = b.shape[1]
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    head = (ctypes.c_void_p(a.data_ptr()), a.stride(0) if m else kp,
            ctypes.c_void_p(b.data_ptr()), b.stride(0), b.stride(1),
            ctypes.c_void_p(scale_a.data_ptr()), _TORCH_CODE[scale_a.dtype],
            ctypes.c_void_p(scale_b.data_ptr()), _TORCH_CODE[scale_b.dtype])
    tail = (ctypes.c_void_p(out.data_ptr()), _TORCH_CODE[out.dtype], out.stride(0) if m else n,
            m, n, kp * 8, _stream(stream))
    if bias is not None:
        bias = bias.to(out.dtype).contiguous()
    if workspace is not None:
        if workspace is True:
            workspace = torch.empty(max(1, gemm_workspace_size(m, n, kp * 8, out.dtype)), dtype=torch.uint8,
                                    device=a.device)
        _check(lib().qo_int4_gemm_ws(*head, ctypes.c_void_p(bias.data_ptr() if bias is not None else None),
                                     *tail[:-1], ctypes.c_void_p(workspace.data_ptr()), workspace.numel(),
                                     tail[-1]))
    elif bias is None:
        _check(lib().qo_int4_gemm(*head, *tail))
    else:
        _check(lib().qo_int4_gemm_bias(*head, ctypes.c_void_p(bias.data_ptr()), *tail))
    return out


def f6_workspace_bytes(m, n, k):
    """``qo_int4_gemm_f6_workspace_bytes``."""
    return int(lib().qo_int4_gemm_f6_workspace_bytes(m, n, k))


def f6_prepare(workspace, m, n, k, a=None, b=None, stream=None):
    """``qo_int4_gemm_f6_prepare``: convert A [M, K/8] and / or B ([K/8, N] or the
    ``W.t()`` view) into ``workspace`` (uint8 device tensor)."""
    if a is not None and a.stride(1) != 1:
        a = a.contiguous()
    if b is not None and b.stride(0) != 1 and b.stride(1) != 1:
        b = b.contiguous()
    _check(lib().qo_int4_gemm_f6_prepare(
        ctypes.c_void_p(a.data_ptr() if a is not None else None), a.stride(0) if a is not None else 0,
        ctypes.c_void_p(b.data_ptr() if b is not None else None), b.stride(0) if b is not None else 0,
        b.stride(1) if b is not None else 0, m, n, k, ctypes.c_void_p(workspace.data_ptr()), workspace.numel(),
        _stream(stream)))


def f6_run(workspace, m, n, k, scale_a, scale_b, out_dtype=torch.float16, out=None, bias=None, stream=None):
    """``qo_int4_gemm_f6_run`` on a prepared ``workspace``; returns out [M, N]."""
    scale_a, scale_b = scale_a.contiguous(), scale_b.contiguous()
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=workspace.device)
    if bias is not None:
        bias = bias.to(out.dtype).contiguous()
    _check(lib().qo_int4_gemm_f6_run(
        ctypes.c_void_p(scale_a.data_ptr()), _TORCH_CODE[scale_a.dtype], ctypes.c_void_p(scale_b.data_ptr()),
        _TORCH_CODE[scale_b.dtype], ctypes.c_void_p(bias.data_ptr() if bias is not None else None),
        ctypes.c_void_p(out.data_ptr()), _TORCH_CODE[out.dtype], out.stride(0), m, n, k,
        ctypes.c_void_p(workspace.data_ptr()), workspace.numel(), _stream(stream)))
    return out


def f6_operand_bytes(rows, k):
    """``qo_int4_gemm_f6_operand_bytes``."""
    return int(lib().qo_int4_gemm_f6_operand_bytes(rows, k))


def f6_convert(src, k, rows_are_columns=False, out=None, stream=None):
    """``qo_int4_gemm_f6_convert``: an operand in the FP6 layout. ``src`` int32
    [rows, K/8] (A, or a [N, K/8] weight whose W.t() is B), or with
    ``rows_are_columns`` a row-major [K/8, N] B. Returns the uint8 tensor."""
    if rows_are_columns:
        rows, rs, ws_ = src.shape[1], src.stride(1), src.stride(0)
    else:
        rows, rs, ws_ = src.shape[0], src.stride(0), src.stride(1)
    n = f6_operand_bytes(rows, k)
    if out is None:
        out = torch.empty(n, dtype=torch.uint8, device=src.device)
    _check(lib().qo_int4_gemm_f6_convert(ctypes.c_void_p(src.data_ptr()), rs, ws_, rows, k,
                                         ctypes.c_void_p(out.data_ptr()), out.numel(), _stream(stream)))
    return out


def w4a4_linear_f6w(x, left, right, weight_f6, out_features, weight_scale, clip_ratio=1.0, bias=None, out=None,
                    codes=None, scales=None, a_workspace=None, stream=None):
    """``qo_w4a4_linear_f6w`` against ``weight_f6`` (``f6_convert(weight, M*N)`` of
    the packed [out, M*N/8] weight). Returns (out, codes, scales)."""
    t, f = x.shape
    if x.stride(1) != 1:
        x = x.contiguous()
    left, right = left.contiguous(), right.contiguous()
    weight_scale = weight_scale.reshape(-1).contiguous()
    m, n = left.shape[0], right.shape[0]
    if codes is None:
        codes = torch.empty((t, f // 8), dtype=torch.int32, device=x.device)
    if scales is None:
        scales = torch.empty((t,), dtype=torch.float32, device=x.device)
    if out is None:
        out = torch.empty((t, out_features), dtype=x.dtype, device=x.device)
    if a_workspace is None:
        a_workspace = torch.empty(max(1, f6_operand_bytes(t, f)), dtype=torch.uint8, device=x.device)
    if bias is not None:
        bias = bias.to(x.dtype).contiguous()
    _check(lib().qo_w4a4_linear_f6w(
        ctypes.c_void_p(x.data_ptr()), _TORCH_CODE[x.dtype], t, x.stride(0) if t else f,
        ctypes.c_void_p(left.data_ptr()), ctypes.c_void_p(right.data_ptr()), m, n, float(clip_ratio),
        ctypes.c_void_p(weight_f6.data_ptr()), weight_f6.numel(), out_features,
        ctypes.c_void_p(weight_scale.data_ptr()), _TORCH_CODE[weight_scale.dtype],
        ctypes.c_void_p(bias.data_ptr() if bias is not None else None),
        ctypes.c_void_p(codes.data_ptr()), ctypes.c_void_p(scales.data_ptr()),
        ctypes.c_void_p(out.data_ptr()), out.stride(0) if t else out_features,
        ctypes.c_void_p(a_workspace.data_ptr()), a_workspace.numel(), _stream(stream)))
    return out, codes, scales


def w4a4_linear(x, left, right, weight, weight_scale, clip_ratio=1.0, bias=None, out=None, codes=None,
                scales=None, stream=None, workspace=None):
    """Call ``qo_w4a4_linear``: x [T, M*N] (float32 / float16 / bfloat16), the packed
    weight int32 [out, M*N/8] (rows may be strided), weight_scale [out], optional
    bias [out] (converted to x's dtype). Returns (out [T, out] in x's dtype, packed
    codes [T, M*N/8], float32 scales [T]). With ``workspace`` (a uint8 device
    tensor, or True to allocate gemm_workspace_size bytes) ``qo_w4a4_linear_ws``."""
    t, f = x.shape
    if x.stride(1) != 1:
        x = x.contiguous()
    left, right = left.contiguous(), right.contiguous()
    if weight.stride(1) != 1:
        weight = weight.contiguous()
    weight_scale = weight_scale.reshape(-1).contiguous()
    m, n = left.shape[0], right.shape[0]
    no = weight.shape[0]
    if codes is None:
        codes = torch.empty((t, f // 8), dtype=torch.int32, device=x.device)
    if scales is None:
        scales = torch.empty((t,), dtype=torch.float32, device=x.device)
    if out is None:
        out = torch.empty((t, no), dtype=x.dtype, device=x.device)
    if bias is not None:
        bias = bias.to(x.dtype).contiguous()
    args = (ctypes.c_void_p(x.data_ptr()), _TORCH_CODE[x.dtype], t, x.stride(0) if t else f,
            ctypes.c_void_p(left.data_ptr()), ctypes.c_void_p(right.data_ptr()), m, n, float(clip_ratio),
            ctypes.c_void_p(weight.data_ptr()), _ld(weight), no,
            ctypes.c_void_p(weight_scale.data_ptr()), _TORCH_CODE[weight_scale.dtype],
            ctypes.c_void_p(bias.data_ptr() if bias is not None else None),
            ctypes.c_void_p(codes.data_ptr()), ctypes.c_void_p(scales.data_ptr()),
            ctypes.c_void_p(out.data_ptr()), out.stride(0) if t else no)
    if workspace is None:
        _check(lib().qo_w4a4_linear(*args, _stream(stream)))
    else:
        if workspace is True:
            workspace = torch.empty(max(1, gemm_workspace_size(t, no, f, x.dtype)), dtype=torch.uint8,
                                    device=x.device)
        _check(lib().qo_w4a4_linear_ws(*args, ctypes.c_void_p(workspace.data_ptr()), workspace.numel(),
                                       _stream(stream)))
    return out, codes, scales


# Byte size of the staging array of qo_w4a4_linear_noalloc (its header's
# QO_LINEAR_NOALLOC_MAX_BYTES).
LINEAR_NOALLOC_MAX_BYTES = 32 * 1024 * 1024


def w4a4_linear_noalloc(x, left, right, weight, weight_scale, clip_ratio=1.0, bias=None, out=None, stream=None):
    """Call ``qo_w4a4_linear_noalloc``: as ``w4a4_linear``, with the activation
    codes and scales staged in the library's per-GPU array instead of caller
    buffers (nothing is allocated except ``out`` when it is not given). Returns
    out [T, out_features] in x's dtype."""
    t, f = x.shape
    if x.stride(1) != 1:
        x = x.contiguous()
    left, right = left.contiguous(), right.contiguous()
    if weight.stride(1) != 1:
        weight = weight.contiguous()
    weight_scale = weight_scale.reshape(-1).contiguous()
    m, n = left.shape[0], right.shape[0]
    no = weight.shape[0]
    if out is None:
        out = torch.empty((t, no), dtype=x.dtype, device=x.device)
    if bias is not None:
        bias = bias.to(x.dtype).contiguous()
    _check(lib().qo_w4a4_linear_noalloc(
        ctypes.c_void_p(x.data_ptr()), _TORCH_CODE[x.dtype], t, x.stride(0) if t else f,
        ctypes.c_void_p(left.data_ptr()), ctypes.c_void_p(right.data_ptr()), m, n, float(clip_ratio),
        ctypes.c_void_p(weight.data_ptr()), _ld(weight), no,
        ctypes.c_void_p(weight_scale.data_ptr()), _TORCH_CODE[weight_scale.dtype],
        ctypes.c_void_p(bias.data_ptr() if bias is not None else None),
        ctypes.c_void_p(out.data_ptr()), out.stride(0) if t else no, _stream(stream)))
    return out


def dequantize_int4(codes, scales, packed_int32=False, out=None, stream=None):
    """Call ``qo_dequantize_int4``; returns float32 [T, F]."""
    codes, scales = codes.contiguous(), scales.contiguous()
    t = codes.shape[0]
    f = codes.shape[1] * (8 if packed_int32 else 1)
    if out is None:
        out = torch.empty((t, f), dtype=torch.float32, device=codes.device)
    _check(lib().qo_dequantize_int4(
        ctypes.c_void_p(codes.data_ptr()), 1 if packed_int32 else 0,
        ctypes.c_void_p(scales.data_ptr()), _TORCH_CODE[scales.dtype], t, f,
        ctypes.c_void_p(out.data_ptr()), _stream(stream)))
    return out


def _ld(t):
    return t.stride(0) if t.dim() == 2 and t.shape[0] > 1 else t.shape[-1]


def pack_int4_to_int32(codes, out=None, stream=None, clamp=False):
    """Call ``qo_pack_int4_to_int32`` (``qo_pack_int4_clamped`` with ``clamp``):
    int8 [rows, F] -> int32 [rows, F/8] (rows may be strided)."""
    assert codes.dtype == torch.int8 and codes.dim() == 2 and codes.stride(1) == 1
    rows, feats = codes.shape
    if out is None:
        out = torch.empty((rows, feats // 8), dtype=torch.int32, device=codes.device)
    pack = lib().qo_pack_int4_clamped if clamp else lib().qo_pack_int4_to_int32
    _check(pack(ctypes.c_void_p(codes.data_ptr()), _ld(codes), rows, feats, ctypes.c_void_p(out.data_ptr()), _ld(out),
                _stream(stream)))
    return out


def unpack_int32_to_int4(words, out=None, stream=None):
    """Call ``qo_unpack_int32_to_int4``: int32 [rows, W] -> int8 [rows, 8W] (rows may be strided)."""
    assert words.dtype == torch.int32 and words.dim() == 2 and words.stride(1) == 1
    rows, nw = words.shape
    if out is None:
        out = torch.empty((rows, 8 * nw), dtype=torch.int8, device=words.device)
    _check(lib().qo_unpack_int32_to_int4(ctypes.c_void_p(words.data_ptr()), _ld(words), rows, nw,
                                         ctypes.c_void_p(out.data_ptr()), _ld(out), _stream(stream)))
    return out


def transpose_int32(x, out=None, stream=None):
    """Call ``qo_transpose_int32``: int32 [R, C] -> contiguous int32 [C, R]."""
    assert x.dtype == torch.int32 and x.dim() == 2 and x.stride(1) == 1
    rows, cols = x.shape
    if out is None:
        out = torch.empty((cols, rows), dtype=torch.int32, device=x.device)
    _check(lib().qo_transpose_int32(ctypes.c_void_p(x.data_ptr()), _ld(x), rows, cols,
                                    ctypes.c_void_p(out.data_ptr()), _ld(out), _stream(stream)))
    return out


_MX_CODE = {"mxfp4": MX_FP4, "mxfp8": MX_FP8}


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr() if t is not None else None)


def _row_stride(t):
    """Stride of a matrix whose rows do not overlap (a single row has one too)."""
    return max(t.stride(0), t.shape[1])


def _unit_rows(t):
    """t, or a copy of it, with unit inner stride."""
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def mx_buffers(tokens, features, fmt, device):
    """Empty codes and scales for [tokens, features] rows (scale rows 16 bytes' multiples apart)."""
    blocks = (features + 31) // 32
    pad = (blocks + 15) // 16 * 16
    codes = (torch.empty((tokens, 16 * blocks), dtype=torch.uint8, device=device) if fmt == "mxfp4" else
             torch.empty((tokens, 32 * blocks), dtype=torch.float8_e4m3fn, device=device))
    return codes, torch.empty((tokens, pad), dtype=torch.uint8, device=device)[:, :blocks]


def mx_quantize(x, fmt="mxfp4", codes=None, scales=None, stream=None):
    """Call ``qo_mx_quantize`` on x [T, F]; returns (codes, scales)."""
    t, f = x.shape
    x = _unit_rows(x)
    if codes is None:
        codes, scales = mx_buffers(t, f, fmt, x.device)
    _check(lib().qo_mx_quantize(_ptr(x), _TORCH_CODE[x.dtype], t, f, _ld(x), _MX_CODE[fmt], _ptr(codes), _ptr(scales),
                                _row_stride(scales), _stream(stream)))
    return codes, scales


def mx_dequantize(codes, scales, features, out_dtype=torch.float32, stream=None):
    """Call ``qo_mx_dequantize``."""
    codes, scales = codes.contiguous(), _unit_rows(scales)
    fmt = MX_FP4 if codes.dtype == torch.uint8 else MX_FP8
    out = torch.empty((codes.shape[0], features), dtype=out_dtype, device=codes.device)
    _check(lib().qo_mx_dequantize(_ptr(codes), _ptr(scales), _row_stride(scales), fmt, codes.shape[0], features, _ptr(out),
                                  _TORCH_CODE[out_dtype], _stream(stream)))
    return out


def rms_norm_mx_quantize(x, weight, eps=1e-6, residual=None, fmt="mxfp8", residual_out=None, stream=None):
    """Call ``qo_rms_norm_mx_quantize``; returns (codes, scales, residual_out or None).
    ``residual_out`` (contiguous) may be a contiguous ``residual`` itself."""
    t, f = x.shape
    x, residual, weight = _unit_rows(x), _unit_rows(residual), weight.contiguous()
    assert residual_out is None or residual_out.is_contiguous()
    codes, scales = mx_buffers(t, f, fmt, x.device)
    if residual is not None and residual_out is None:
        residual_out = torch.empty((t, f), dtype=x.dtype, device=x.device)
    _check(lib().qo_rms_norm_mx_quantize(_ptr(x), _ptr(residual), _TORCH_CODE[x.dtype], t, f, _ld(x),
                                         _ld(residual) if residual is not None else 0, _ptr(weight),
                                         _TORCH_CODE[weight.dtype], float(eps), _MX_CODE[fmt], _ptr(codes),
                                         _ptr(scales), _row_stride(scales), _ptr(residual_out), _stream(stream)))
    return codes, scales, residual_out


def swiglu_mx_quantize(gate_up, fmt="mxfp8", stream=None):
    """Call ``qo_swiglu_mx_quantize`` on [T, 2 F]; returns (codes, scales)."""
    t, f = gate_up.shape[0], gate_up.shape[1] // 2
    gate_up = _unit_rows(gate_up)
    codes, scales = mx_buffers(t, f, fmt, gate_up.device)
    _check(lib().qo_swiglu_mx_quantize(_ptr(gate_up), _TORCH_CODE[gate_up.dtype], t, f, _ld(gate_up), _MX_CODE[fmt],
                                       _ptr(codes), _ptr(scales), _row_stride(scales), _stream(stream)))
    return codes, scales


def mx_gemm_workspace_size(m, n, k, fmt):
    """``qo_mx_gemm_workspace_size``."""
    return int(lib().qo_mx_gemm_workspace_size(m, n, k, _MX_CODE[fmt]))


def mx_gemm(a, a_scales, b, b_scales, bias=None, out_dtype=torch.bfloat16, out=None, stream=None, workspace=None):
    """Call ``qo_mx_gemm``: a (uint8 or float8_e4m3fn codes) [M, ..], b uint8 [N, K/2], rows 16-byte
    aligned; bias is taken in the output dtype. ``workspace``: a uint8 device tensor, or True to allocate one."""
    m, n, blocks = a.shape[0], b.shape[0], a_scales.shape[1]
    if workspace is True:
        need = mx_gemm_workspace_size(m, n, 32 * blocks, "mxfp4" if a.dtype == torch.uint8 else "mxfp8")
        workspace = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    assert out.stride(1) == 1 or n == 1
    a, a_scales, b, b_scales = (_unit_rows(t) for t in (a, a_scales, b, b_scales))
    if bias is not None:
        bias = bias.to(out.dtype).contiguous()
    _check(lib().qo_mx_gemm(_ptr(a), _ld(a), MX_FP4 if a.dtype == torch.uint8 else MX_FP8, _ptr(a_scales), _row_stride(a_scales),
                            _ptr(b), _ld(b), _ptr(b_scales), _row_stride(b_scales), _ptr(bias), _ptr(out),
                            _TORCH_CODE[out.dtype], _ld(out), m, n, 32 * blocks, _ptr(workspace),
                            workspace.numel() if workspace is not None else 0, _stream(stream)))
    return out


def kv4_struct(cache):
    """``qo_kv4_cache`` of the three tensors (``quant_ops_amd.KV4Cache``)."""
    k, v, params = cache
    assert k.is_contiguous() and v.is_contiguous() and params.is_contiguous()
    return KV4Struct(k.data_ptr(), v.data_ptr(), params.data_ptr(), k.shape[0], k.shape[2], k.shape[1], 2 * k.shape[3])


def _heads(x):
    return None if x is None else ctypes.byref(HeadsStruct(x.data_ptr(), x.stride(0), x.stride(1)))


def kv4_append(cache, k, v, slots, positions=None, cos=None, sin=None, q=None, interleaved=False, stream=None):
    """Call ``qo_kv4_append``; returns the rotated q or None."""
    k, v, q = _unit_rows(k), _unit_rows(v), _unit_rows(q)
    slots = slots.contiguous()
    positions, cos, sin = (None if t is None else t.contiguous() for t in (positions, cos, sin))
    out = None if q is None else torch.empty(tuple(q.shape), dtype=q.dtype, device=q.device)
    _check(lib().qo_kv4_append(ctypes.byref(kv4_struct(cache)), _heads(q), _heads(k), _heads(v), _TORCH_CODE[k.dtype],
                               k.shape[0], 0 if q is None else q.shape[1], _ptr(slots), _ptr(positions), _ptr(cos), _ptr(sin),
                               0 if cos is None else cos.shape[0], 0 if cos is None else 2 * cos.shape[1], int(interleaved),
                               _ptr(out), _stream(stream)))
    return out


def kv4_read(cache, slots, out_dtype=torch.float32, stream=None):
    """Call ``qo_kv4_read``; returns (k, v)."""
    slots = slots.contiguous()
    shape = (slots.shape[0], cache[0].shape[1], 2 * cache[0].shape[3])
    k, v = (torch.empty(shape, dtype=out_dtype, device=slots.device) for _ in range(2))
    _check(lib().qo_kv4_read(ctypes.byref(kv4_struct(cache)), _ptr(slots), slots.shape[0], _ptr(k), _ptr(v),
                             _TORCH_CODE[out_dtype], _stream(stream)))
    return k, v


def kv4_attention_workspace_size(cache, dtype, tokens, q_heads, table_width, sequences, has_starts=False, window=0):
    """``qo_kv4_attention_workspace_size``."""
    return int(lib().qo_kv4_attention_workspace_size(ctypes.byref(kv4_struct(cache)), _TORCH_CODE[dtype], tokens, q_heads, table_width, sequences,
                                                     int(has_starts), window))


def kv4_attention(q, cache, page_table, lengths, scale, q_starts=None, window=0, out=None, workspace=None, stream=None):
    """Call ``qo_kv4_attention``. ``workspace``: a uint8 device tensor, or True to allocate one."""
    q, page_table, lengths = _unit_rows(q), _unit_rows(page_table), lengths.contiguous()
    batch, width = page_table.shape
    if workspace is True:
        need = kv4_attention_workspace_size(cache, q.dtype, q.shape[0], q.shape[1], width, batch, q_starts is not None, window)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    if out is None:
        out = torch.empty(tuple(q.shape), dtype=q.dtype, device=q.device)
    assert out.is_contiguous() and (q_starts is None or q_starts.is_contiguous())
    _check(lib().qo_kv4_attention(ctypes.byref(kv4_struct(cache)), _heads(q), _TORCH_CODE[q.dtype], q.shape[0], q.shape[1],
                                  _ptr(page_table), _ld(page_table), width, _ptr(lengths), _ptr(q_starts), batch, float(scale),
                                  window, _ptr(out), _ptr(workspace), workspace.numel() if workspace is not None else 0,
                                  _stream(stream)))
    return out
