"""GPU tests of attention over the 4-bit cache with scores that lie so far apart that each row is its largest one's value."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_cases import HALF_STEP, U
from kv4_grid import on_a_grid
from oracle import kv4_reference as ok

pytestmark = pytest.mark.gpu

CASES = [   # few rows, and many in tiles of either size
    ([90, 33], 4, 2, 64, 16, 1, 0),
    ([150, 21], 8, 1, 128, 32, 2, 0),
    ([90, 70], 2, 1, 256, 16, 10, 0),
    ([3000, 500], 4, 1, 128, 64, 1, 0),      # several workgroups to a sequence
    ([99, 140], 3, 1, 96, 32, 33, 50),
    ([230, 150], 2, 1, 128, 16, 100, 0),
    ([2000], 4, 1, 128, 64, 20, 0),          # several workgroups to a tile
    ([1500], 4, 1, 64, 64, 40, 0),
]


def one_value_a_row(gpu, q, cache, table, lengths, window, scale):
    """The weights are 1 (equal ones share) and 0: the output is off by a weight's rounding, the middle's two products and
    sums, the division's rounding and its own."""
    out, mag, _ = ok.attention(q, cache, table, lengths, scale, None, window)
    got = qo.kv4_attention(q.to(gpu), qo.KV4Cache(*(t.to(gpu) for t in cache)), table.to(gpu), lengths.to(gpu), scale=scale,
                           window=window).cpu().double()
    assert bool(torch.isfinite(got).all())
    weight = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -22
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    off = (got - out).abs() / ((HALF_STEP[q.dtype] + 2 * U) * (out.abs() + weight * mag) + (weight + 6 * U) * mag + tiny + 1e-300)
    print(f"[gpu-kv4] {float(off.max()):.3f} of the bound", flush=True)
    assert float(off.max()) <= 1.0


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("scale", [2.0 ** 14, 2.0 ** 22, 1e9, 1e30])
def test_large_scales(gpu, scale, case, dtype):
    """Steps of 2^7 and more between scores up to 2^30 and far above."""
    print(f"[gpu-kv4] far {scale} {case} {dtype}", flush=True)
    q, cache, table, lengths, window = on_a_grid(case, 8.0)
    one_value_a_row(gpu, q.to(dtype), cache, table, lengths, window, scale)
