"""GPU tests of the microscaled RMS norm's arithmetic: y is the formula's value rounded once to
float32, whatever the row's sum of squares."""
import pytest
import torch

import quant_ops_amd as qo
from oracle import mx_reference as om
from test_gpu_mx import FMTS, _check_near, _rows

pytestmark = pytest.mark.gpu

# One rounding to float32; the sum, the root and the products are held in 64 bits, whose
# roundings (2^-53 each, a few thousand of them) are far below the rest.
ONCE = 2.0 ** -24 * (1 + 2.0 ** -12)

# both sides of the lines between the kernel's variants, and rows that are read twice
LENGTHS = [32, 96, 512, 1000, 4096, 4104, 8192, 8200, 16384, 24576, 28672, 32768, 32776, 70000, 4099, 33001]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("feats", LENGTHS)
def test_codes_beside_a_tie(gpu, feats, fmt):
    """Weights that put y two units of float32 below the middle between two codes, on rows whose
    squares a running float32 sum loses: of each eight values one is 1, the others' squares lie
    under half its last bit."""
    g = torch.Generator().manual_seed(feats)
    h = 2.0 ** -12 * (0.8 + 0.15 * torch.rand(1, feats, generator=g))
    h[:, ::8] = 1.0
    grid = om.GRID4 if fmt == "mxfp4" else torch.arange(0, 127).to(torch.uint8).view(torch.float8_e4m3fn).double()
    middles = (grid[1:] + grid[:-1]) / 2
    target = middles[torch.randint(8 if fmt == "mxfp8" else 0, len(middles), (feats,), generator=g)]
    target[::32] = middles[-1]   # holds the block's exponent at 0
    r = 1 / torch.sqrt(h.double().square().mean() + 1e-6)
    w = (target * (1 - 2.0 ** -23) / (h[0].double() * r)).float()
    print(f"[gpu-mx-norm] {feats} {fmt}", flush=True)
    codes, scales = qo.rms_norm_mx_quantize(h.to(gpu), w.to(gpu), 1e-6, fmt=fmt)
    torch.cuda.synchronize()
    _check_near(om.rms_norm(h, w, torch.tensor(1e-6).double())[1], ONCE, fmt, codes, scales)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("feats", [100, 4096, 8192, 40000])
def test_squares_past_float32(gpu, feats, dtype, fmt):
    """Rows whose squares leave float32 at either end: their norm is a row of ordinary size.
    (2^-70 with eps 0: squares of 2^-140; 2^90: of 2^180, a sum's mean past 2^127 as well.)"""
    x = torch.randn(6, feats, generator=torch.Generator().manual_seed(feats))
    for rows, power in ((slice(0, 2), 90), (slice(2, 4), -70), (slice(4, 6), 122)):
        x[rows] *= 2.0 ** power
    x = x.to(dtype)
    w = torch.linspace(0.5, 1.5, feats)
    print(f"[gpu-mx-norm] large and small rows, {feats} {dtype} {fmt}", flush=True)
    codes, scales = qo.rms_norm_mx_quantize(x.to(gpu), w.to(gpu), 0.0, fmt=fmt)
    torch.cuda.synchronize()
    _check_near(om.rms_norm(x, w, 0.0)[1], ONCE, fmt, codes, scales)


@pytest.mark.parametrize("with_residual", (False, True))
def test_rows_of_activations(gpu, with_residual):
    """Ordinary rows, at the bound of one rounding."""
    x = _rows(700, 4096, torch.bfloat16, 1)
    res = _rows(700, 4096, torch.bfloat16, 2) if with_residual else None
    w = torch.linspace(-1.5, 1.5, 4096)
    got = qo.rms_norm_mx_quantize(x.to(gpu), w.to(gpu), residual=None if res is None else res.to(gpu))
    torch.cuda.synchronize()
    h = x.float() if res is None else x.float() + res.float()
    _check_near(om.rms_norm(h, w, torch.tensor(1e-6).double())[1], ONCE, "mxfp8", got[0], got[1])
