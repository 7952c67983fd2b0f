"""GPU tests of attention over the 4-bit cache for sequences of many rows with keys, queries and values that are not
centred or not of one size: outlier channels, offset keys, large queries, small values. All types are held to
kv4_cases.bound, which counts no rounding of keys or values: the codes are multiplied exactly."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_cases import batch, check
from test_kv4_cpu import DTYPES

pytestmark = pytest.mark.gpu

SHAPES = [   # lengths, query heads, KV heads, head_dim, page, queries each, window
    ([230, 150], 2, 1, 128, 16, 100, 0),     # 200 rows a sequence
    ([260, 190], 4, 2, 64, 64, 90, 120),
    ([230, 150], 3, 1, 96, 16, 70, 0),
    ([200, 65], 3, 1, 128, 64, 33, 0),       # 99
    ([150, 130], 3, 1, 256, 32, 40, 0),
    ([150, 130], 6, 2, 192, 16, 30, 70),
]
SEVERAL = ("two channels by 20", "two channels by 50", "one channel biased", "offset by 100", "offset by 1000", "large queries",
           "values of 2^-14", "values of 2^-17", "values of 2^-20", "values of 2^10")


def _inputs(kind, shape, dtype):
    lengths, heads, kv, dim, page, queries, window = shape
    g = torch.Generator().manual_seed(dim + len(kind))
    table, pages = batch(g, lengths, page)
    cache = qo.kv4_cache(pages, page, kv, dim, device="cpu")
    total = sum(lengths)
    k, v = torch.randn(total, kv, dim, generator=g), torch.randn(total, kv, dim, generator=g)
    q = 1.5 * torch.randn(queries * len(lengths), heads, dim, generator=g)
    channels = [3, dim - 7]
    if kind.startswith("two channels"):
        by = float(kind.split()[-1])
        k[..., channels] += by
        q[..., channels] *= by / 4
    elif kind == "one channel biased":
        k[..., 5] += 60.0
        q[..., 5] += 60.0
    elif kind.startswith("offset"):
        k += float(kind.split()[-1])
    elif kind == "large queries":
        q *= 8.0
    else:
        v *= 2.0 ** float(kind.split("^")[1])
    at = 0
    for b, n in enumerate(lengths):
        t = torch.arange(n)
        qo.kv4_append(cache, k[at:at + n], v[at:at + n], table[b].long()[t // page] * page + t % page)
        at += n
    return q.to(dtype), cache, table, torch.tensor(lengths, dtype=torch.int32), window


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", SEVERAL)
@pytest.mark.parametrize("shape", SHAPES)
def test_prompts(gpu, shape, kind, dtype):
    print(f"[gpu-kv4] prompt {shape} {kind} {dtype}", flush=True)
    q, cache, table, lengths, window = _inputs(kind, shape, dtype)
    got = qo.kv4_attention(q.to(gpu), qo.KV4Cache(*(t.to(gpu) for t in cache)), table.to(gpu), lengths.to(gpu), window=window)
    worst = check(q, got, cache, table, lengths, q.shape[2] ** -0.5, None, window)
    print(f"[gpu-kv4] {worst:.3f} of the bound", flush=True)
