"""Host forms of the microscaled operators where the ordinary cases do not reach."""
import pytest
import torch

import quant_ops_amd as qo
from oracle import mx_reference as om

FMTS = ("mxfp4", "mxfp8")


@pytest.mark.parametrize("fmt", FMTS)
def test_norm_of_squares_past_float32(fmt):
    """Rows whose squares leave float32 at either end; y is the formula's value rounded once, but
    for the two 64-bit computations' own roundings."""
    x = torch.randn(6, 100, generator=torch.Generator().manual_seed(1))
    for rows, power in ((slice(0, 2), 90), (slice(2, 4), -70), (slice(4, 6), 122)):
        x[rows] *= 2.0 ** power
    w = torch.linspace(0.5, 1.5, 100)
    codes, scales = qo.rms_norm_mx_quantize(x, w, 0.0, fmt=fmt)
    q, byte = om.quantize(om.rms_norm(x, w, 0.0)[1].float(), fmt)
    assert torch.equal(scales.long(), byte) and torch.equal(om.code_values(codes), q)


def test_host_refusals_equal_the_gpu():
    """What the GPU operators refuse, host tensors are refused for too (lists of test_gpu_mx.py's refusals)."""
    x = torch.zeros(4, 64)
    b, sb = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    b8 = torch.zeros(8, 64).to(torch.float8_e4m3fn)
    w = torch.ones(64)
    bad = [
        lambda: qo.mx_quantize(x.double()),
        lambda: qo.mx_quantize(x.int()),
        lambda: qo.mx_dequantize(b, sb[:, :1]),
        lambda: qo.mx_dequantize(b.int(), sb),
        lambda: qo.mx_dequantize(b, sb.int()),
        lambda: qo.mx_dequantize(b, sb, out_dtype=torch.float64),
        lambda: qo.rms_norm_mx_quantize(x, w[:63]),
        lambda: qo.rms_norm_mx_quantize(x, w[:1]),
        lambda: qo.rms_norm_mx_quantize(x, w.double()),
        lambda: qo.rms_norm_mx_quantize(x, w, residual=x.half()),
        lambda: qo.swiglu_mx_quantize(x.double()),
        lambda: qo.mx_matmul(b, sb, b[:, :16], sb[:, :1]),
        lambda: qo.mx_matmul(b, sb[:4], b, sb),
        lambda: qo.mx_matmul(b.float(), sb, b, sb),
        lambda: qo.mx_matmul(b, sb, b8, sb),
        lambda: qo.mx_matmul(b, sb, b, sb, bias=torch.zeros(7)),
        lambda: qo.mx_matmul(b, sb, b, sb, bias=torch.zeros(1)),
        lambda: qo.mx_matmul(b, sb, b, sb, out_dtype=torch.float64),
        lambda: qo.mx_matmul(b, sb.float(), b, sb),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was accepted")


def test_bias_of_any_shape_of_n_elements():
    """As on the GPU: a bias holds N elements."""
    a, sa = qo.mx_quantize(torch.randn(3, 64, generator=torch.Generator().manual_seed(2)), "mxfp8")
    b, sb = qo.mx_quantize(torch.randn(8, 64, generator=torch.Generator().manual_seed(3)))
    bias = torch.arange(8.0)
    assert torch.equal(qo.mx_matmul(a, sa, b, sb, bias=bias.view(8, 1)), qo.mx_matmul(a, sa, b, sb, bias=bias))
