"""GPU tests of both store forms of the microscaled dequantizer: non-temporal 16-byte pieces where the
output is 16-byte aligned and its rows are whole pieces, ordinary ones elsewhere."""
import pytest
import torch

from oracle import mx_reference as om
from quant_ops_amd import capi
from test_gpu_mx import DTYPES, FMTS, _operand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,feats", [(3, 64), (5, 4096), (2, 100), (4, 36), (3, 33)])
@pytest.mark.parametrize("offset", (0, 1))
def test_output_pointers(gpu, offset, tokens, feats, dtype, fmt):
    """Whole rows of pieces at an aligned pointer and one element past it; other lengths. Nothing
    is written before or behind the output."""
    codes, scales = _operand(tokens, -(-feats // 32), fmt, feats, 100, 150)
    codes, dscales = codes.to(gpu), scales.to(gpu)
    raw = torch.full((tokens * feats + 24,), 7.0, dtype=dtype, device=gpu)
    at = 8 + offset
    out = raw[at:at + tokens * feats]
    assert raw.data_ptr() % 16 == 0
    print(f"[gpu-mx-dequantize] {tokens} x {feats} {dtype} {fmt} + {offset}", flush=True)
    capi._check(capi.lib().qo_mx_dequantize(
        capi._ptr(codes), capi._ptr(dscales), dscales.shape[1], capi.MX_FP4 if fmt == "mxfp4" else capi.MX_FP8, tokens,
        feats, capi._ptr(out), capi._TORCH_CODE[dtype], capi._stream(None)))
    torch.cuda.synchronize()
    assert torch.equal(out.cpu().view(tokens, feats), om.values(codes, scales)[:, :feats].to(dtype))
    assert bool((raw[:at] == 7.0).all()) and bool((raw[at + tokens * feats:] == 7.0).all())
