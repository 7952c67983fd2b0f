"""The microscaled operators from their definition, in 64 bits (for tests; no
counterpart in the reference).

Written apart from the package: exponents from ``math.frexp``-style arithmetic
on float64, FP4 rounding by comparison with the midpoints of its grid, FP8 by
the spacing of the e4m3 grid.
"""
import torch

EMAX = {"mxfp4": 2, "mxfp8": 8}
GRID4 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
MID4 = (GRID4[1:] + GRID4[:-1]) / 2


def _exponent(v):
    """floor(log2 v) of positive float64 values."""
    return torch.frexp(v)[1] - 1


def scale_bytes(top, fmt):
    """Scale byte of each largest magnitude (float64)."""
    e = _exponent(torch.where((top > 0) & torch.isfinite(top), top, 1.0)) - EMAX[fmt]
    e = torch.where(top == 0, -127, e).clamp(-127, 127)
    return torch.where(torch.isfinite(top), e + 127, 255)


def blocks_of(y):
    """[T, F] float64 -> [T, B, 32] padded with zeros."""
    t, f = y.shape
    b = -(-f // 32)
    v = torch.zeros(t, 32 * b, dtype=torch.float64)
    v[:, :f] = y
    return v.view(t, b, 32)


def round_codes(q, fmt):
    """q (float64) rounded to the format's nearest value, ties to the even code, saturated."""
    mag = q.abs()
    if fmt == "mxfp4":
        lo, hi = torch.bucketize(mag, MID4), torch.bucketize(mag, MID4, right=True)   # differ at a tie
        v = GRID4[torch.where(lo % 2 == 0, lo, hi)]
    else:
        unit = torch.ldexp(torch.ones_like(mag), _exponent(torch.where(mag > 0, mag, 1.0)).clamp(min=-6) - 3)
        v = (torch.round(mag / unit) * unit).clamp(max=448)
    return torch.copysign(v, q)


def quantize(y, fmt):
    """Values of the codes [T, B, 32] (float64, signed zeros kept) and scale bytes [T, B] of y [T, F]."""
    v = blocks_of(y.double())
    top = torch.where(torch.isnan(v).any(2), float("inf"), v.abs().amax(2))
    byte = scale_bytes(top, fmt)
    ok = (byte < 255)[:, :, None]
    q = torch.where(ok, v, 0.0) / torch.ldexp(torch.ones_like(top), byte.clamp(max=254) - 127)[:, :, None]
    return round_codes(q, fmt), byte


def code_values(codes):
    """Values of codes: uint8 [T, 16 B] or float8_e4m3fn [T, 32 B] -> float64 [T, B, 32]."""
    codes = codes.cpu()
    if codes.dtype == torch.uint8:
        nib = torch.stack((codes & 15, codes >> 4), 2).flatten(1).long()
        v = GRID4[nib & 7]
        v = torch.where(nib >= 8, -v, v)
    else:
        v = codes.float().double()
    return v.view(v.shape[0], v.shape[1] // 32, 32)


def values(codes, scales):
    """What codes and scales stand for, float64 [T, 32 B]."""
    byte = scales.cpu().long()
    s = torch.where(byte == 255, float("nan"), torch.ldexp(torch.ones_like(byte, dtype=torch.float64), byte - 127))
    return (code_values(codes) * s[:, :, None]).flatten(1)


def rms_norm(x, weight, eps, residual=None):
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * weight.double()


def swiglu(gate_up):
    g, u = gate_up.double().chunk(2, 1)
    return g / (1 + torch.exp(-g)) * u


def matmul(a, a_scales, b, b_scales):
    """The product and the sum of its terms' magnitudes, float64 [M, N]."""
    x, y = values(a, a_scales), values(b, b_scales)
    return x @ y.t(), x.abs() @ y.abs().t()
