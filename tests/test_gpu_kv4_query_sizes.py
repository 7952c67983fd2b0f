"""GPU tests of attention over the 4-bit cache with queries of any size that float32 and bfloat16 hold."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_grid import on_a_grid
from test_gpu_kv4_far_scores import CASES as FAR, one_value_a_row
from test_kv4_cpu import make

pytestmark = pytest.mark.gpu

WIDE = (torch.float32, torch.bfloat16)
CASES = [   # few rows, and many in tiles of either size
    ([90, 33], 4, 2, 64, 16, 1, 0),
    ([150, 21], 8, 1, 128, 32, 2, 0),
    ([90, 70], 2, 1, 256, 16, 10, 0),
    ([99, 140], 3, 1, 96, 32, 33, 50),
    ([230, 150], 2, 1, 128, 16, 100, 0),
]


def _run(gpu, q, cache, table, lengths, window, scale):
    got = qo.kv4_attention(q.to(gpu), qo.KV4Cache(*(t.to(gpu) for t in cache)), table.to(gpu), lengths.to(gpu), scale=scale, window=window)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("power", [-110, -60, 60, 110, 123])
def test_a_power_of_two_may_stand_in_the_scale(gpu, power, case, dtype):
    """Queries times a power of two and the scale divided by it: the same scores, to the last bit. |q| < 8 leaves
    2^123 q finite, and 2^-110 q keeps its bits (those below 2^-16 in q are 0 here)."""
    print(f"[gpu-kv4] power {power} {case} {dtype}", flush=True)
    q, cache, table, lengths, _, window = make(case, torch.float32)
    q = ((q.clamp(-7.9, 7.9) * 4096).round() / 4096).to(dtype)
    scale = 0.125
    want = _run(gpu, q, cache, table, lengths, window, scale)
    got = _run(gpu, (q.double() * 2.0 ** power).to(dtype), cache, table, lengths, window, scale * 2.0 ** -power)
    assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("case", FAR)
@pytest.mark.parametrize("power,scale", [(114, 0.125), (119, 1.0), (100, 2.0 ** 14), (-100, 2.0 ** 127)])
def test_scores_next_to_the_largest_number(gpu, power, scale, case, dtype):
    """Queries and scales that bring scores next to the largest that float32 holds, or their product back."""
    print(f"[gpu-kv4] next to {power} {scale} {case} {dtype}", flush=True)
    q, cache, table, lengths, window = on_a_grid(case, 4.0)
    one_value_a_row(gpu, (q.double() * 2.0 ** power).to(dtype), cache, table, lengths, window, scale)
