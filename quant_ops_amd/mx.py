"""Microscaled (OCP MX) formats: quantize, dequantize, the product with 4-bit
weights, and the RMS norm and SwiGLU gate that quantize their result.

Along a row, 32 consecutive values share a scale 2^e, held as the byte e + 127
(255: NaN), and are coded as ``"mxfp4"`` (FP4 e2m1) or ``"mxfp8"`` (FP8 e4m3).
A row of F values has B = ceil(F / 32) blocks, the last padded with zeros:

* mxfp4 codes: uint8 [T, 16 B], two per byte, the even value in the low bits;
* mxfp8 codes: float8_e4m3fn [T, 32 B];
* scales: uint8 [T, B]; those made on the GPU stand a multiple of 16 bytes apart
  by rows, as the product of many rows reads them (others are copied).

e = floor(log2(largest magnitude)) - 2 (mxfp4) or - 8 (mxfp8), at least -127;
codes are v / 2^e rounded to nearest even, saturated at 6 or 448. A block that
holds a NaN or an infinity gets the scale byte 255 and zero codes, and reads
back (and multiplies) as NaN.

GPU tensors use the HIP kernels through ``torch.ops.quant_ops``; if the HIP
library is not loaded they raise. Host tensors run the formulas in PyTorch.
All of it is for inference: codes carry no gradient. None of these functions
has a counterpart in the reference.
"""
from typing import Optional, Tuple

import torch

from . import _loader

BLOCK = 32
_EMAX = {"mxfp4": 2, "mxfp8": 8}
_FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _emax(fmt):
    if fmt not in _EMAX:
        raise ValueError(f'fmt must be "mxfp4" or "mxfp8", got {fmt!r}')
    return _EMAX[fmt]


def _rows(x):
    return x if x.dim() == 2 else x[None] if x.dim() == 1 else x.flatten(0, -2)


def _like(t, x):
    """[T, ...] rows as x's leading dimensions."""
    return t if x.dim() == 2 else t.reshape(*x.shape[:-1], t.shape[1])


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _check(ok, message):
    """Host tensors are refused where the GPU operators refuse them."""
    if not ok:
        raise ValueError(message)


def _check_float(t, name):
    _check(t.dtype in _FLOATS, f"{name} dtype must be float32, float16 or bfloat16, got {t.dtype}")


def _check_codes(codes, scales, name):
    _check(codes.dtype in (torch.uint8, torch.float8_e4m3fn),
           f"{name} must be uint8 (FP4 codes) or float8_e4m3fn (FP8 codes), got {codes.dtype}")
    _check(scales.dtype == torch.uint8, f"{name}'s scales must be uint8, got {scales.dtype}")
    _check(codes.shape == (scales.shape[0], scales.shape[1] * (BLOCK // 2 if codes.dtype == torch.uint8 else BLOCK)),
           f"{name} {tuple(codes.shape)} and its scales {tuple(scales.shape)} do not match")


def _check_out(out_dtype):
    _check(out_dtype in _FLOATS, f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")


def _quantize_pytorch(y, fmt):
    """Codes and scales of float32 rows y [T, F]."""
    emax = _emax(fmt)
    tokens, feats = y.shape
    blocks = -(-feats // BLOCK)
    v = torch.nn.functional.pad(y.float(), (0, BLOCK * blocks - feats)).view(tokens, blocks, BLOCK)
    top = v.abs().amax(2) if blocks else v.new_zeros(tokens, 0)
    e = torch.where(top == 0, -127, torch.frexp(top)[1] - 1 - emax).clamp(-127, 127)
    bad = ~torch.isfinite(top)
    # in float64: 2^e and v / 2^e are exact at every exponent
    q = torch.where(bad[:, :, None], 0.0, v.double() / torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)[:, :, None])
    scales = torch.where(bad, 255, e + 127).to(torch.uint8)
    if fmt == "mxfp8":
        return q.clamp(-448, 448).float().to(torch.float8_e4m3fn).flatten(1), scales
    mag = q.abs()
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    near = (torch.round(mag / step) * step).clamp(max=6)
    grid = torch.tensor(_FP4_VALUES, dtype=torch.float64, device=y.device)
    code = (torch.searchsorted(grid, near) + 8 * torch.signbit(q)).to(torch.uint8).flatten(1)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def _values_pytorch(codes, scales):
    """float32 [T, 32 B] of codes and scales."""
    if codes.dtype == torch.uint8:
        table = torch.tensor(_FP4_VALUES + tuple(-v for v in _FP4_VALUES), device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), 2).long()].flatten(1)
    else:
        v = codes.float()
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    s = torch.where(scales == 255, float("nan"), s).float()
    return (v.view(*s.shape, BLOCK) * s[:, :, None]).flatten(1)


# The operators' overloads, looked up once (a lookup costs as much as a check). A library
# built before these operators lacks them: the package imports with it all the same.
_OPS = ("mx_quantize", "mx_dequantize", "rms_norm_mx_quantize", "add_rms_norm_mx_quantize", "swiglu_mx_quantize", "mx_matmul")
_op = {name: getattr(torch.ops.quant_ops, name).default for name in _OPS
       if _loader.KERNELS_AVAILABLE and hasattr(torch.ops.quant_ops, name)}


def _gpu(name):
    _loader.require_kernels(name)
    if name not in _op:
        raise RuntimeError(f"{name}: the loaded library ({_loader.TORCH_LIB_PATH}) does not have it; "
                           "rebuild with python -m quant_ops_amd._build")
    return _op[name]


def mx_quantize(x: torch.Tensor, fmt: str = "mxfp4") -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of x [..., F] (float32 / float16 / bfloat16)."""
    if x.is_cuda and x.dim() == 2:
        return _gpu("mx_quantize")(x, fmt)
    rows = _rows(x)
    if x.is_cuda:
        codes, scales = _gpu("mx_quantize")(rows, fmt)
    else:
        _check_float(x, "input")
        codes, scales = _quantize_pytorch(rows, fmt)
    return _like(codes, x), _like(scales, x)


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, features: Optional[int] = None,
                  out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of codes and scales, [..., features] in out_dtype (each rounded
    once); features defaults to the padded row length."""
    if codes.is_cuda and codes.dim() == 2:
        return _gpu("mx_dequantize")(codes, scales, features, out_dtype)
    q, s = _rows(codes), _rows(scales)
    if codes.is_cuda:
        out = _gpu("mx_dequantize")(q, s, features, out_dtype)
    else:
        _check_codes(q, s, "codes")
        _check_out(out_dtype)
        feats = BLOCK * s.shape[1] if features is None else features
        assert -(-feats // BLOCK) == s.shape[1], f"features ({feats}) must fill the {s.shape[1]} blocks of a row"
        out = _values_pytorch(q, s)[:, :feats].to(out_dtype)
    return _like(out, codes)


def rms_norm_mx_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                         residual: Optional[torch.Tensor] = None, fmt: str = "mxfp8") -> Tuple[torch.Tensor, ...]:
    """RMS norm of x (+ residual), quantized: ``(codes, scales)``, and with a
    residual ``(codes, scales, x + residual)``.

    h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, both rounded once to
    float32; the sum is returned rounded once to x's dtype. x and residual [..., F] of one
    dtype, weight [F] of any of the three.
    """
    if x.is_cuda and x.dim() == 2:
        if residual is None:
            return _gpu("rms_norm_mx_quantize")(x, weight, eps, fmt)
        return _gpu("add_rms_norm_mx_quantize")(x, residual, weight, eps, fmt)
    rows = _rows(x)
    res = None if residual is None else _rows(residual)
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} must have x's shape {tuple(x.shape)}")
    if x.is_cuda:
        got = (_gpu("rms_norm_mx_quantize")(rows, weight, eps, fmt) if res is None else
               _gpu("add_rms_norm_mx_quantize")(rows, res, weight, eps, fmt))
    else:
        _check_float(x, "x")
        _check_float(weight, "weight")
        _check(weight.shape == rows.shape[1:], f"weight must hold one value per feature ({rows.shape[1]}), got {tuple(weight.shape)}")
        _check(res is None or res.dtype == x.dtype, "residual must have x's dtype")
        h = rows.float() if res is None else rows.float() + res.float()
        wide = h.double()   # squares leave float32 where h does not
        got = _quantize_pytorch((wide / torch.sqrt(wide.square().mean(1, keepdim=True) + eps) * weight.double()).float(), fmt)
        if res is not None:
            got = (*got, h.to(x.dtype))
    return tuple(_like(t, x) for t in got)


def swiglu_mx_quantize(gate_up: torch.Tensor, fmt: str = "mxfp8") -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of silu(g) * u in float32, gate_up [..., 2 F] holding the
    gate g and then its factor u."""
    if gate_up.is_cuda and gate_up.dim() == 2:
        return _gpu("swiglu_mx_quantize")(gate_up, fmt)
    rows = _rows(gate_up)
    if gate_up.is_cuda:
        codes, scales = _gpu("swiglu_mx_quantize")(rows, fmt)
    else:
        _check_float(gate_up, "gate_up")
        _check(rows.shape[1] % 2 == 0, f"gate_up must hold two halves, got {tuple(gate_up.shape)}")
        g, u = rows.float().chunk(2, 1)
        codes, scales = _quantize_pytorch(g / (1 + torch.exp(-g)) * u, fmt)
    return _like(codes, gate_up), _like(scales, gate_up)


def mx_matmul(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor,
              bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T (+ bias)`` of the values that the codes stand for, float32 sums of
    exact products, rounded once to out_dtype.

    a [..., K] mxfp4 or mxfp8 codes with a_scales [..., K/32]; b the weight's
    mxfp4 codes [N, K/2] with b_scales [N, K/32]; bias [N] (taken in out_dtype).
    """
    if a.is_cuda and a.dim() == 2:
        return _gpu("mx_matmul")(a, a_scales, b, b_scales, bias, out_dtype)
    q, s = _rows(a), _rows(a_scales)
    if a.is_cuda:
        out = _gpu("mx_matmul")(q, s, b, b_scales, bias, out_dtype)
    else:
        _check_codes(q, s, "a")
        _check_codes(b, b_scales, "b")
        _check(b.dtype == torch.uint8, f"b must be uint8 (FP4 codes), got {b.dtype}")
        _check(b_scales.shape[1] == s.shape[1], f"b's scales {tuple(b_scales.shape)} do not match a's {s.shape[1]} blocks")
        _check(bias is None or bias.numel() == b.shape[0], f"bias must hold N ({b.shape[0]}) elements")
        _check_out(out_dtype)
        out = _values_pytorch(q, s) @ _values_pytorch(b, b_scales).t()
        out = (out if bias is None else out + bias.to(out_dtype).float().reshape(-1)).to(out_dtype)
    return _like(out, a)
