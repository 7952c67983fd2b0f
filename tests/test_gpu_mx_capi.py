"""GPU tests of the ctypes calls of the microscaled operators on tensors that the C interface does not
take as they are: they are copied, as the other calls of ``capi`` do."""
import pytest
import torch

import quant_ops_amd as qo
from quant_ops_amd import capi
from test_gpu_mx import FMTS, _operand, _rows

pytestmark = pytest.mark.gpu


def _same(got, want):
    assert all(torch.equal(g.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8)) for g, w in zip(got, want) if g is not None)


@pytest.mark.parametrize("fmt", FMTS)
def test_strided_rows_and_weights(gpu, fmt):
    wide = _rows(6, 512, torch.bfloat16, 1).to(gpu)
    x, res, w = wide[:, ::2], wide[:, 1::2], torch.linspace(-1, 2, 512, device=gpu)[::2]
    assert x.stride(1) == 2
    _same(capi.mx_quantize(x, fmt), qo.mx_quantize(x.contiguous(), fmt))
    _same(capi.rms_norm_mx_quantize(x, w, residual=res, fmt=fmt),
          qo.rms_norm_mx_quantize(x.contiguous(), w.contiguous(), residual=res.contiguous(), fmt=fmt))
    _same(capi.swiglu_mx_quantize(x, fmt), qo.swiglu_mx_quantize(x.contiguous(), fmt))
    codes, scales = qo.mx_quantize(wide, fmt)
    half = codes.shape[1] // 2
    _same([capi.mx_dequantize(codes[:, :half], scales[:, :8], 256)], [qo.mx_dequantize(codes[:, :half].contiguous(), scales[:, :8].contiguous())])


@pytest.mark.parametrize("out_dtype", (torch.float32, torch.bfloat16))
def test_bias_of_another_type(gpu, out_dtype):
    """A bias is taken in the output's type, whatever its own, and strided ones by their elements."""
    (a, sa), (b, sb) = _operand(5, 4, "mxfp8", 1), _operand(40, 4, "mxfp4", 2)
    a, sa, b, sb = (t.to(gpu) for t in (a, sa, b, sb))
    for bias in (torch.linspace(-4, 4, 40, device=gpu), torch.linspace(-4, 4, 40, device=gpu).half(),
                 torch.linspace(-4, 4, 80, device=gpu).bfloat16()[::2]):
        _same([capi.mx_gemm(a, sa, b, sb, bias=bias, out_dtype=out_dtype)], [qo.mx_matmul(a, sa, b, sb, bias=bias, out_dtype=out_dtype)])
