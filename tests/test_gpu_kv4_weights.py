"""GPU tests of attention over the 4-bit cache for few rows a sequence: 16-bit outputs are the rounded values of float32
ones, not of sums of weights that were rounded to 16 bits first."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_cases import U
from kv4_grid import on_a_grid
from oracle import kv4_reference as ok

pytestmark = pytest.mark.gpu

LENGTHS = [3, 4, 5, 6, 7, 9, 12, 20]
CASES = [(LENGTHS, heads, 2, dim, 16, queries, 0) for dim in (64, 96, 128, 192, 256) for heads, queries in ((8, 1), (16, 1), (16, 2))]


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("case", CASES)
def test_outputs_are_rounded_once(gpu, case, dtype):
    """Each output is a rounding of a value no further from the exact one than float32 leaves it, for scores that
    float32 holds: a weight counts twice (numerator and denominator), with three roundings in units of its exponent, at
    most 16 here, two of its own and 2^-22 for two parts in 16 bits; two middles and products; a rounding for each
    of a lane's 16 tokens and the joins of the lanes, waves and parts, and the division's."""
    print(f"[gpu-kv4] weights {case} {dtype}", flush=True)
    q, cache, table, lengths, _ = on_a_grid(case, 4.0)
    q = q.to(dtype)
    scale = 1 / case[3]
    out, mag, big = ok.attention(q, cache, table, lengths, scale)
    assert float(big.max()) < 11                     # 16 in powers of two
    got = qo.kv4_attention(q.to(gpu), qo.KV4Cache(*(t.to(gpu) for t in cache)), table.to(gpu), lengths.to(gpu), scale=scale).cpu()
    off = (2 * (3 * 16 * U + 2 * U + 2.0 ** -22) + (4 + 16 + 12 + 1) * U) * mag
    low, high = (out - off).to(dtype), (out + off).to(dtype)
    outside = (got < low) | (got > high)
    print(f"[gpu-kv4] {int(outside.sum())} of {outside.numel()} outside", flush=True)
    assert not bool(outside.any())
