"""GPU tests of attention over the 4-bit cache beside memory that holds anything: what stands in places that no
query sees has no say in any bit of the outputs."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_cases import check
from test_kv4_cpu import DTYPES, make

pytestmark = pytest.mark.gpu

CASES = [   # lengths, query heads, KV heads, head_dim, page, queries each (a list: ragged, with two rows behind), window
    ([230, 150], 2, 1, 128, 16, 100, 60),      # 200 rows a sequence
    ([230, 150], 2, 1, 64, 64, 100, 0),
    ([99, 140], 3, 1, 64, 64, 33, 50),         # 99
    ([99, 140], 3, 1, 96, 32, 33, 0),
    ([150, 90], 3, 1, 256, 32, 33, 0),
    ([150, 390], 2, 2, 192, 16, [80, 70], 100),
    ([150, 21], 6, 2, 96, 16, 1, 0),           # few
    ([90, 333], 8, 1, 128, 32, 3, 70),
    ([77, 31], 4, 1, 256, 64, 2, 0),
    ([3000, 10], 4, 1, 128, 64, 1, 1000),
]


def _seen(cache, table, lengths, starts, queries, window):
    """Truth values [pages, page_size] of the slots that some query sees."""
    pages, _, size, _ = cache.k_codes.shape
    seen = torch.zeros(pages, size, dtype=torch.bool)
    for b, length in enumerate(lengths.tolist()):
        n = queries if starts is None else int(starts[b + 1] - starts[b])
        t = torch.arange(max(0, length - n + 1 - window) if window else 0, length)
        seen[table[b].long()[t // size], t % size] = True
    return seen


def _fill(cache, places, params, codes):
    """The cache with the parameters params [pages, page_size, 2, heads, 2] and the codes' bytes at the places."""
    k, v, p = (t.clone() for t in cache)
    page, place = places.nonzero(as_tuple=True)
    k[page, :, place] = codes
    v[page, :, place // 16, :, place % 16] = codes
    p[page, :, :, place // 16, :, place % 16] = params[page, place]
    return qo.KV4Cache(k, v, p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_unseen_places_have_no_say(gpu, case, dtype):
    print(f"[gpu-kv4] unseen {case} {dtype}", flush=True)
    q, cache, table, lengths, starts, window = make(case, dtype)
    pages, heads, size, _ = cache.k_codes.shape
    unseen = ~_seen(cache, table, lengths, starts, case[5], window)
    g = torch.Generator().manual_seed(1)
    shape = (pages, size, 2, heads, 2)
    bits = torch.randint(0, 1 << 16, shape, generator=g)
    bits = torch.where(bits & 0x7C00 == 0x7C00, bits & ~0x4000, bits)       # finite
    finite = torch.where(bits > 0x7FFF, bits - (1 << 16), bits).to(torch.int16).view(torch.float16)
    most = torch.where(torch.rand(shape, generator=g) < 0.5, -65504.0, 65504.0).half()

    def run(cache, table):
        got = qo.kv4_attention(q.to(gpu), qo.KV4Cache(*(t.to(gpu) for t in cache)), table.to(gpu), lengths.to(gpu),
                               q_starts=None if starts is None else starts.to(gpu), window=window)
        torch.cuda.synchronize()
        return got

    clean = run(_fill(cache, unseen, torch.zeros(shape, dtype=torch.float16), 0), table)
    check(q, clean, cache, table, lengths, q.shape[2] ** -0.5, starts, window)
    # entries of the table past a sequence's tokens name pages that hold garbage as well
    elsewhere = torch.where(table < 0, pages - 1, table)
    for params in (finite, most, torch.full(shape, 65504.0, dtype=torch.float16),
                   torch.full(shape, float("inf"), dtype=torch.float16), torch.full(shape, float("nan"), dtype=torch.float16)):
        assert torch.equal(run(_fill(cache, unseen, params, 0xFF), elsewhere), clean)
