"""GPU tests of the microscaled product's sums where large terms cancel: what is left has to
be right to float32 sums in every kernel, with every output type."""
import pytest
import torch

import quant_ops_amd as qo
from oracle import mx_reference as om
from test_gpu_mx import _check_product
from test_gpu_mx_tiles import CASES, OUTS, STREAM

pytestmark = pytest.mark.gpu


def _cancelling(m, n, blocks, seed):
    """FP8 rows of a in two halves along K: of each eight codes one is large (256 .. 448) and the
    others small (2^-4 .. 1); the second half has the same large ones negated and zeros
    besides. b's halves are equal. So the large terms cancel, and out is the small terms' sum."""
    g = torch.Generator().manual_seed(seed)
    half = blocks // 2
    small = torch.randint(3 << 3, 8 << 3, (m, 32 * half), generator=g)
    large = torch.randint(15 << 3, (15 << 3) + 7, (m, 4 * half), generator=g)
    at = torch.arange(0, 32 * half, 8) + torch.randint(0, 8, (4 * half,), generator=g)
    sign = 128 * torch.randint(0, 2, (m, 32 * half), generator=g)
    first = small + sign
    first[:, at] = large + sign[:, at]
    second = torch.zeros_like(first)
    second[:, at] = first[:, at] ^ 128
    middle = torch.zeros(m, 32 * (blocks - 2 * half), dtype=torch.long)
    a = torch.cat((first, middle, second), 1).to(torch.uint8).view(torch.float8_e4m3fn)
    sa = torch.full((m, blocks), 127, dtype=torch.uint8)
    b = torch.randint(0, 256, (n, 16 * half), generator=g).to(torch.uint8)
    b = torch.cat((b, torch.zeros(n, 16 * (blocks - 2 * half), dtype=torch.uint8), b), 1)
    sb = torch.full((n, blocks), 127, dtype=torch.uint8)
    return a, sa, b, sb


def _check_float32_sums(out, a, sa, b, sb):
    """|out - exact| against one rounding to the output type and the bound of _check_product for
    float32 sums alone (2^-22 of the terms' magnitudes and 2^-23 of them a k-step)."""
    want, mag = om.matmul(a, sa, b, sb)
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[out.dtype]
    steps = 2 * -(-sa.shape[1] // 4) + 16
    bound = unit * want.abs() + (1 + unit) * (2.0 ** -22 + 2.0 ** -23 * steps) * mag
    off = (out.cpu().double() - want).abs() > bound
    assert not bool(off.any()), f"{int(off.sum())} of {off.numel()} outputs off"


SIZES = [(m, n, blocks, tile, parts) for m, n, blocks, fmt, tile, parts in CASES if fmt == "mxfp8" and 1 < blocks < 64]
SIZES += [(m, n, blocks, "stream", 1) for m, n, blocks in STREAM if 1 < blocks < 130]
SIZES += [(18, 97, 193, "64", 8), (77, 520, 129, "64", 4)]


@pytest.mark.parametrize("m,n,blocks,tile,parts", SIZES)
def test_cancelling_terms(gpu, m, n, blocks, tile, parts):
    a, sa, b, sb = _cancelling(m, n, blocks, m + n)
    print(f"[gpu-mx-sums] {m} x {n} x {32 * blocks}: {tile} in {parts}", flush=True)
    for out_dtype in OUTS:
        out = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), out_dtype=out_dtype)
        torch.cuda.synchronize()
        _check_float32_sums(out, a, sa, b, sb)
        _check_product(out, a, sa, b, sb)
