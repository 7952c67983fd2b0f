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
