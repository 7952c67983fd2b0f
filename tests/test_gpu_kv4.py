"""GPU tests of the 4-bit key/value cache against its definition in 64 bits.

Appending and reading are exact: every border between codes is decided in 64 bits, so the
cache equals the oracle's byte for byte. Attention is held to the bound of kv4_cases.bound."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_cases import angles, batch, check, random_cache, vectors
from oracle import kv4_reference as ok
from quant_ops_amd import capi
from test_kv4_cpu import CASES, DTYPES, _same, check_refused, make, refusals

pytestmark = pytest.mark.gpu


def _say(msg):
    print(f"[gpu-kv4] {msg}", flush=True)


def _to(cache, device):
    return qo.KV4Cache(*(t.to(device) for t in cache))


def test_refusals(gpu):
    check_refused(refusals(gpu))


# ------------------------------------------------------------- append and read
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot,interleaved,page,tokens,heads,kv", [
    (64, 64, False, 16, 1, 1, 1), (64, 32, True, 32, 33, 5, 2), (96, 96, False, 16, 7, 4, 4), (96, 8, True, 64, 50, 3, 1),
    (128, 128, False, 64, 100, 8, 2), (128, 64, True, 16, 17, 2, 2), (192, 192, True, 16, 9, 3, 3), (192, 56, False, 128, 31, 1, 1),
    (256, 256, False, 16, 23, 4, 2), (256, 128, True, 32, 8, 2, 1)])
def test_append_and_read(gpu, dim, rot, interleaved, page, tokens, heads, kv, dtype):
    _say(f"append {dim} {rot} {interleaved} {page} {tokens} {dtype}")
    g = torch.Generator().manual_seed(dim + rot + tokens)
    pages = -(-tokens // page) * 2 + 1
    start = random_cache(g, pages, page, kv, dim)
    want = tuple(t.clone() for t in start)
    row = vectors(g, tokens, heads + 2 * kv, dim).to(dtype)
    q, k, v = row[:, :heads], row[:, heads:heads + kv], row[:, heads + kv:]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 8:
        slots[3], slots[7], slots[8] = -1, pages * page, 1 << 40
    pos = torch.randint(0, 60, (tokens,), generator=g)
    cos, sin = angles(60, rot)
    cache, d = _to(start, gpu), row.to(gpu)
    got = qo.kv4_append(cache, d[:, heads:heads + kv], d[:, heads + kv:], slots.to(gpu), positions=pos.to(gpu), cos=cos.to(gpu),
                        sin=sin.to(gpu), q=d[:, :heads], interleaved=interleaved)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), ok.turn(q, pos, cos, sin, interleaved).float().to(dtype))
    for which, x in enumerate((ok.turn(k, pos, cos, sin, interleaved).float(), v.float())):
        c, s, lo = ok.store(x)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                ok.put(want, which, slot, c[t], s[t], lo[t])
    assert _same([t.cpu() for t in cache], want)
    for out_dtype in DTYPES:
        for which, x in enumerate(qo.kv4_read(cache, slots.to(gpu), out_dtype)):
            assert x.dtype == out_dtype
            for t, slot in enumerate(slots.tolist()):
                row = ok.read(want, which, slot, out_dtype) if 0 <= slot < pages * page else torch.zeros(kv, dim, dtype=out_dtype)
                assert torch.equal(x[t].cpu(), row)


def _both(gpu, x, v, slots, page=16, pages=2, **turn):
    """The same append on the host and the GPU: both caches, and the queries' results."""
    host = qo.kv4_cache(pages, page, x.shape[1], x.shape[2], device="cpu")
    dev = qo.kv4_cache(pages, page, x.shape[1], x.shape[2], device=gpu)
    a = qo.kv4_append(host, x, v, slots, **turn)
    b = qo.kv4_append(dev, x.to(gpu), v.to(gpu), slots.to(gpu), **{n: t.to(gpu) if torch.is_tensor(t) else t for n, t in turn.items()})
    torch.cuda.synchronize()
    return host, dev, a, b


def test_vectors_at_the_edges(gpu):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(9, 1, 64, generator=g)
    x[0], x[1] = 3.25, 0.0
    x[2, 0, 5], x[3, 0, 63], x[4, 0, 0] = float("nan"), float("inf"), -float("inf")
    x[5] *= 1e30
    x[6] *= 1e-30
    x[7] = torch.arange(64) * 0.25 - 3
    x[8] = 1000 + 0.001 * x[8]
    host, dev, _, _ = _both(gpu, x, -x, torch.arange(9))
    assert _same(host, [t.cpu() for t in dev])
    for dtype in DTYPES:
        for a, b in zip(qo.kv4_read(host, torch.arange(9), dtype), qo.kv4_read(dev, torch.arange(9, device=gpu), dtype)):
            assert torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b.cpu(), 7.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(gpu, dtype):
    """Vectors whose every value lies on a border between two codes, or a float32 step beside one."""
    n = torch.arange(128)
    rows = []
    for s, lo in ((1.0, 0.0), (0.5, -3.0), (2.0 ** -10, 1.0), (0.0999755859375, -0.5)):   # fp16 values
        tie = lo + s * (n % 15 + 0.5)
        for step in (0, 1, -1):
            near = torch.nextafter(tie.float(), torch.full_like(tie, step * 1e9)) if step else tie.float()
            near[0], near[1] = lo, lo + 15 * s
            rows.append(near)
    x = torch.stack(rows)[:, None].to(dtype)
    host, dev, _, _ = _both(gpu, x, x.flip(2), torch.arange(len(rows)))
    c, s, lo = ok.store(x.float())
    want = tuple(t.clone() for t in host)
    for t in range(len(rows)):
        ok.put(want, 0, t, c[t], s[t], lo[t])
    assert _same(host, want) and _same(host, [t.cpu() for t in dev])


def test_position_outside_the_table(gpu):
    x = torch.ones(4, 1, 64)
    cos, sin = angles(4, 32)
    host, dev, a, b = _both(gpu, x, x, torch.arange(4), positions=torch.tensor([1, 4, -1, 1 << 40]), cos=cos, sin=sin, q=x)
    assert _same(host, [t.cpu() for t in dev])
    assert torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b.cpu(), 7.0)) and torch.isnan(b[1:, :, :32]).all()


def test_large_prefill_equals_the_host(gpu):
    g = torch.Generator().manual_seed(11)
    x = vectors(g, 2000, 6, 128).bfloat16()
    cos, sin = angles(4000, 128)
    slots = torch.randperm(40 * 64, generator=g)[:2000].sort()[0]   # runs of neighbours
    host, dev, a, b = _both(gpu, x[:, 2:4], x[:, 4:], slots, page=64, pages=40, positions=torch.arange(2000) + 1999, cos=cos, sin=sin,
                            q=x[:, :2])
    assert torch.equal(a, b.cpu()) and _same(host, [t.cpu() for t in dev])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv,interleaved,first", [(64, 19, 7, False, 33), (128, 19, 7, True, 65), (192, 11, 9, False, 2), (96, 40, 4, True, 64)])
def test_many_heads_equal_the_host(gpu, dim, heads, kv, interleaved, first, dtype):
    """Several heads to a workgroup, the last groups not full; a run of slots that starts inside a word, with holes; values
    of few bits, so that many lie on a border between codes."""
    _say(f"many heads {dim} {heads} {kv} {first} {dtype}")
    g = torch.Generator().manual_seed(dim + heads)
    tokens = 2100
    x = (torch.randint(-60, 61, (tokens, heads + 2 * kv, dim), generator=g) / 8).to(dtype)
    slots = torch.arange(tokens) + first
    slots[::97] = -1
    cos, sin = angles(tokens, dim)
    host, dev, a, b = _both(gpu, x[:, heads:heads + kv], x[:, heads + kv:], slots, page=64, pages=40, positions=torch.arange(tokens),
                            cos=cos, sin=sin, q=x[:, :heads], interleaved=interleaved)
    assert torch.equal(a, b.cpu()) and _same(host, [t.cpu() for t in dev])


def test_other_strides(gpu):
    """Heads before tokens, values at a stride of two, one row for all tokens, offsets of one element."""
    g = torch.Generator().manual_seed(12)
    for make_view in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                      lambda t: torch.stack((t, t), 3).flatten(2)[..., ::2],
                      lambda t: t[:1].expand(t.shape),
                      lambda t: torch.cat((torch.zeros(1, dtype=t.dtype), t.flatten()))[1:].view(t.shape)):
        x = vectors(g, 20, 2, 96).half()
        cos, sin = angles(20, 96)
        kw = dict(positions=torch.arange(20), cos=cos, sin=sin)
        y = make_view(x)
        dev = y.to(gpu) if y.stride() == x.stride() else make_view(x.to(gpu))
        host, ref = qo.kv4_cache(2, 16, 2, 96, device="cpu"), qo.kv4_cache(2, 16, 2, 96, device=gpu)
        a = qo.kv4_append(host, y, y, torch.arange(20), q=y, **kw)
        kw = {n: t.to(gpu) for n, t in kw.items()}
        b = qo.kv4_append(ref, dev, dev, torch.arange(20, device=gpu), q=dev, **kw)
        assert torch.equal(a, b.cpu()) and _same(host, [t.cpu() for t in ref])


# ------------------------------------------------------------------- attention
def _run(gpu, q, cache, table, lengths, starts=None, window=0, scale=None):
    got = qo.kv4_attention(q.to(gpu), _to(cache, gpu), table.to(gpu), lengths.to(gpu), scale=scale,
                           q_starts=None if starts is None else starts.to(gpu), window=window)
    torch.cuda.synchronize()
    return got


def _check(gpu, q, cache, table, lengths, starts=None, window=0):
    got = _run(gpu, q, cache, table, lengths, starts, window)
    assert got.dtype == q.dtype and got.shape == q.shape
    worst = check(q, got, cache, table, lengths, q.shape[2] ** -0.5, starts, window)
    _say(f"{worst:.3f} of the bound")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_attention(gpu, case, dtype):
    _say(f"attention {case} {dtype}")
    _check(gpu, *make(case, dtype))


GPU_CASES = [
    ([700], 8, 2, 128, 64, 1, 0),
    ([2100, 1, 600], 4, 1, 128, 16, 1, 0),
    ([1500, 900], 2, 2, 64, 128, 2, 0),
    ([1300], 16, 1, 256, 32, 1, 0),
    ([1200, 77], 3, 1, 192, 16, 4, 300),
    ([600], 5, 1, 96, 64, 13, 0),
    ([330, 1000, 64], 8, 2, 128, 32, [70, 33, 64], 0),
    ([128, 260], 4, 4, 64, 16, [128, 129], 0),
    ([300, 5], 16, 1, 96, 256, [100, 1], 40),
    ([400], 7, 1, 128, 16, 90, 0),
    ([140] * 70, 2, 1, 64, 16, [1] * 35 + [0] * 20 + [2] * 15, 0),   # more sequences than a wave has lanes
    ([200, 330], 4, 2, 128, 16, 50, 0),            # more than 64 rows a sequence
    ([500], 8, 1, 64, 64, 40, 0),
    ([257, 64, 1], 6, 2, 96, 32, [130, 64, 1], 0),
    ([300], 3, 1, 192, 16, 100, 130),
    ([150, 90], 5, 1, 256, 16, 30, 0),
    ([100], 2, 1, 128, 16, 150, 0),
    ([700, 20], 2, 2, 128, 32, [300, 20], 200),
    ([900], 4, 1, 128, 64, 200, 0),                # seven tiles of 128 rows
    ([640], 2, 1, 64, 32, 320, 100),
    ([500, 450, 333], 3, 1, 128, 16, [300, 129, 43], 0),
    ([3], 1, 1, 256, 16, 3, 0),
    ([2], 2, 1, 128, 16, 40, 0),       # queries before the first token
    ([4000, 70], 4, 1, 64, 64, 1, 0),  # many parts
]


# Every kernel of every head size: waves of 4, 8 and 16 rows, prompts in tiles of 128 and 256.
EVERY_KERNEL = [c for dim in (64, 96, 128, 192, 256) for c in (
    ([150, 21], 6, 2, dim, 16, 1, 0),
    ([99, 140], 6, 1, dim, 32, 1, 70),
    ([77, 200, 31], 6, 1, dim, 16, [9, 4, 3], 0),
    ([90, 333], 8, 1, dim, 32, 3, 0),
    ([200, 65], 3, 1, dim, 64, 33, 0),
    ([190, 260], 3, 1, dim, 16, [110, 90], 0),
)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", GPU_CASES + EVERY_KERNEL)
def test_attention_more(gpu, case, dtype):
    _say(f"attention {case} {dtype}")
    _check(gpu, *make(case, dtype))


def test_masked_places_may_hold_anything(gpu):
    q, cache, table, lengths, _, _ = make(([37], 2, 1, 64, 16, 4, 10), torch.float32)
    for t in list(range(37, 48)) + list(range(0, 24)) + [35]:
        page, place = int(table[0, t // 16]), t % 16
        cache.params[page, :, :, place // 16, :, place % 16] = float("nan") if t % 2 else float("inf")
    got = _run(gpu, q, cache, table, lengths, window=10)
    assert not torch.isnan(got[:2]).any() and torch.isnan(got[2:]).all()
    check(q, got, cache, table, lengths, 64 ** -0.5, None, 10)


def test_masked_values_only(gpu):
    """A token whose value alone is NaN, seen by the later queries of a tile and not by the earlier."""
    q, cache, table, lengths, _, _ = make(([100], 4, 1, 128, 16, 8, 0), torch.bfloat16)
    page, place = int(table[0, 6]), 96 % 16
    cache.params[page, 1, :, place // 16, :, place % 16] = float("nan")      # token 96; queries stand at 92 .. 99
    got = _run(gpu, q, cache, table, lengths)
    assert not torch.isnan(got[:4]).any() and torch.isnan(got[4:]).all()
    check(q, got, cache, table, lengths, 128 ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_places_in_prompts(gpu, dtype):
    """The same for sequences of many rows: garbage behind the last token and before the window, a token whose
    value is NaN, one whose key is, a page outside the cache, and NaN and infinite queries."""
    q, cache, table, lengths, _, _ = make(([230, 150], 2, 1, 128, 16, 100, 60), dtype)   # queries from 130 and 50 on
    for b, t in ((0, 170), (1, 100)):
        cache.params[int(table[b, t // 16]), 1 - b, :, t % 16 // 16, 0, t % 16] = float("nan")
    for t in list(range(0, 70)) + list(range(230, 240)):
        cache.params[int(table[0, t // 16]), :, :, 0, :, t % 16] = float("inf")
    table[1, 9] = -1                                        # tokens 144 ..
    q[20, 1, 7], q[30, 0, 100] = float("nan"), -float("inf")
    got = _run(gpu, q, cache, table, lengths, window=60)
    i = torch.arange(200)
    p = torch.where(i < 100, 130 + i, i - 50)
    bad = torch.where(i < 100, (p >= 170) & (p < 230), (p >= 100) & (p < 160))[:, None].repeat(1, 2)
    bad[20, 1] = bad[30, 0] = True
    assert torch.equal(torch.isnan(got).any(2).cpu(), bad) and torch.equal(torch.isnan(got).all(2).cpu(), bad)
    q[20, 1, 7] = q[30, 0, 100] = 0.0
    got = _run(gpu, q, cache, table, lengths, window=60)
    check(q, got, cache, table, lengths, 128 ** -0.5, None, 60)


def test_bad_pages_and_lengths(gpu):
    q, cache, table, lengths, _, _ = make(([40, 40, 40, 40, -3], 2, 1, 64, 16, 1, 0), torch.float32)
    table[0, 1], table[1, 2], lengths[2] = -1, cache.k_codes.shape[0], 16 * table.shape[1] + 1
    got = _run(gpu, q, cache, table, lengths)
    assert [bool(torch.isnan(got[i]).all()) for i in range(5)] == [True, True, True, False, False]
    assert not torch.isnan(got[3:]).any() and not got[4].any()
    check(q, got, cache, table, lengths, 64 ** -0.5)


def test_starts_that_do_not_ascend_stay_inside(gpu):
    """Whatever q_starts holds, only rows of the output are written."""
    q, cache, table, lengths, _, _ = make(([40, 40, 40], 2, 1, 64, 16, 4, 0), torch.float32)
    for starts in ([0, 9, 3, 12], [5, 2, 1, 0], [0, 100, -7, 1 << 30], [0, 0, 0, 0], [-4, 6, 6, 12]):
        out = torch.full((q.shape[0] + 64,) + tuple(q.shape[1:]), 3.0, device=gpu)
        capi.kv4_attention(q.to(gpu), _to(cache, gpu), table.to(gpu), lengths.to(gpu), 0.125,
                           q_starts=torch.tensor(starts, dtype=torch.int32, device=gpu), out=out[32:32 + q.shape[0]])
        torch.cuda.synchronize()
        assert bool((out[:32] == 3).all()) and bool((out[32 + q.shape[0]:] == 3).all())


def test_empty_calls(gpu):
    cache = qo.kv4_cache(2, 16, 2, 64, device=gpu)
    none = torch.zeros(0, 2, 64, device=gpu)
    qo.kv4_append(cache, none, none, torch.zeros(0, dtype=torch.int64, device=gpu))
    k, v = qo.kv4_read(cache, torch.zeros(0, dtype=torch.int64, device=gpu))
    assert k.shape == v.shape == (0, 2, 64)
    i32 = dict(dtype=torch.int32, device=gpu)
    assert qo.kv4_attention(none, cache, torch.zeros(0, 2, **i32), torch.zeros(0, **i32)).shape == none.shape
    rows = torch.ones(3, 2, 64, device=gpu)
    got = qo.kv4_attention(rows, cache, torch.zeros(0, 2, **i32), torch.zeros(0, **i32), q_starts=torch.zeros(1, **i32))
    assert not got.any()
    assert not qo.kv4_attention(rows, cache, torch.zeros(3, 0, **i32), torch.zeros(3, **i32)).any()
    assert torch.isnan(qo.kv4_attention(rows, cache, torch.zeros(3, 0, **i32), torch.ones(3, **i32))).all()
    nothing = qo.kv4_cache(0, 16, 2, 64, device=gpu)
    qo.kv4_append(nothing, rows, rows, torch.arange(3, device=gpu))
    assert not qo.kv4_read(nothing, torch.arange(3, device=gpu))[0].any()
    assert torch.isnan(qo.kv4_attention(rows, nothing, torch.zeros(3, 1, **i32), torch.ones(3, **i32))).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_of_any_size(gpu, dtype):
    """Rows of zeros, very large and very small queries, and NaN and infinities, which stay in their row."""
    q, cache, table, lengths, _, _ = make(([90] * 7, 4, 2, 64, 16, 1, 0), dtype)
    q[0] = 0.0
    q[1] *= 1000.0
    q[2] *= 2.0 ** -14
    q[3, :, ::2] *= 2.0 ** -12
    q[4, 1, 3], q[5, 0, 9], q[5, 2, 9] = float("nan"), float("inf"), -float("inf")
    got = _run(gpu, q, cache, table, lengths)
    bad = torch.zeros(7, 4, dtype=torch.bool)
    bad[4, 1] = bad[5, 0] = bad[5, 2] = True
    assert torch.equal(torch.isnan(got).all(2).cpu(), bad) and torch.equal(torch.isnan(got).any(2).cpu(), bad)
    q[4:6] = 1.0
    got = _run(gpu, q, cache, table, lengths)
    check(q, got, cache, table, lengths, 64 ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** 10])
def test_values_of_any_size(gpu, dtype, size):
    """Scales at either end of fp16, growing from step to step."""
    g = torch.Generator().manual_seed(3)
    table, pages = batch(g, [400], 16)
    cache = random_cache(g, pages, 16, 2, 128)
    for i, page in enumerate(table[0].tolist()):
        cache.params[page, 1] = (cache.params[page, 1].float() * size * 2.0 ** (i % 5)).half()
    q = torch.randn(1, 4, 128, generator=g).to(dtype)
    _check(gpu, q, cache, table, torch.tensor([400], dtype=torch.int32))


def test_tokens_far_below_the_largest(gpu):
    """One token far above 3000 others of equal weight, whose sum still counts."""
    g = torch.Generator().manual_seed(4)
    table, pages = batch(g, [3000], 64)
    cache = random_cache(g, pages, 64, 1, 64)
    cache.k_codes.zero_()
    cache.params[:, 0] = 0.0
    cache.params[:, 0, :, :, 1] = -1.0
    page = int(table[0, 0])
    cache.params[page, 0, :, 0, 1, 5] = 1.0
    q = torch.full((1, 1, 64), 1.0)                      # scores -8, and 8 for token 5: weights e^-16
    for dtype in DTYPES:
        _check(gpu, q.to(dtype), cache, table, torch.tensor([3000], dtype=torch.int32))


def test_split_and_whole_agree(gpu):
    """The same call with a workspace (parts joined) and without, and a workspace with garbage in it."""
    for case in (([5000], 4, 1, 128, 64, 1, 0), ([3000, 10], 2, 2, 64, 16, [3, 1], 0)):
        q, cache, table, lengths, starts, window = (t.to(gpu) if torch.is_tensor(t) else t for t in make(case, torch.float32))
        cache = _to(cache, gpu)
        need = capi.kv4_attention_workspace_size(cache, q.dtype, q.shape[0], q.shape[1], table.shape[1], table.shape[0], starts is not None)
        assert need > 0
        ws = torch.full((need,), 255, dtype=torch.uint8, device=gpu)
        a = capi.kv4_attention(q, cache, table, lengths, 0.1, q_starts=starts, workspace=ws)
        b = capi.kv4_attention(q, cache, table, lengths, 0.1, q_starts=starts)
        c = capi.kv4_attention(q, cache, table, lengths, 0.1, q_starts=starts, workspace=ws[:need - 16])
        torch.cuda.synchronize()
        for out in (a, b, c):
            check(q.cpu(), out, [t.cpu() for t in cache], table.cpu(), lengths.cpu(), 0.1, None if starts is None else starts.cpu())
        assert torch.equal(b, c)


def test_same_call_same_bits(gpu):
    q, cache, table, lengths, starts, window = make(([2000, 300], 8, 2, 128, 16, [40, 7], 0), torch.bfloat16)
    first = _run(gpu, q, cache, table, lengths, starts)
    for _ in range(3):
        assert torch.equal(first, _run(gpu, q, cache, table, lengths, starts))


def test_strided_queries_and_tables(gpu):
    q, cache, table, lengths, _, _ = make(([90, 200, 33], 4, 2, 96, 16, 2, 0), torch.float16)
    want = _run(gpu, q, cache, table, lengths)
    d = [t.to(gpu) for t in (q, table, lengths)]
    c = _to(cache, gpu)
    for view in (lambda t: torch.cat((t, t), 1)[:, :t.shape[1]], lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.stack((t, t), -1).flatten(-2)[..., ::2], lambda t: torch.cat((t, t), 2)[..., :t.shape[2]]):
        assert torch.equal(want, qo.kv4_attention(view(d[0]), c, d[1], d[2]))
    wide = torch.full((3, 50), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = d[1]
    for t in (wide[:, :table.shape[1]], d[1].t().contiguous().t(), torch.stack((d[1], d[1]), 2).flatten(1)[:, ::2]):
        assert torch.equal(want, qo.kv4_attention(d[0], c, t, d[2]))
    # a wider table may be shared out differently: held to the bound
    check(q, qo.kv4_attention(d[0], c, wide, torch.stack((d[2], d[2]), 1)[:, 0]), cache, table, lengths, 96 ** -0.5)


def test_one_page_for_two_sequences(gpu):
    """A shared prefix: the same pages in two rows of the table."""
    q, cache, table, lengths, _, _ = make(([90, 90], 2, 1, 64, 16, 1, 0), torch.bfloat16)
    table[1, :3] = table[0, :3]
    _check(gpu, q, cache, table, lengths)


def test_offsets_past_32_bits(gpu):
    """A cache whose parts pass 4 GiB."""
    heads, dim, page = 4, 128, 64
    pages = (1 << 32) // (heads * page * dim // 2) + 40
    cache = qo.kv4_cache(pages, page, heads, dim, device=gpu)
    assert cache.k_codes.numel() > 1 << 32 and cache.v_codes.numel() > 1 << 32
    g = torch.Generator().manual_seed(6)
    small = qo.kv4_cache(3, page, heads, dim, device="cpu")
    x = vectors(g, 150, heads, dim).bfloat16()
    slots = torch.arange(150)
    qo.kv4_append(small, x, -x, slots)
    far = torch.tensor([pages - 1, pages - 30, 1])
    at = far[slots // page] * page + slots % page
    qo.kv4_append(cache, x.to(gpu), -x.to(gpu), at.to(gpu))
    for a, b in zip(qo.kv4_read(cache, at.to(gpu)), qo.kv4_read(small, slots)):
        assert torch.equal(a.cpu(), b)
    q = torch.randn(1, 8, dim, generator=g).bfloat16()
    lengths = torch.tensor([150], dtype=torch.int32)
    got = qo.kv4_attention(q.to(gpu), cache, far[None].int().to(gpu), lengths.to(gpu))
    check(q, got, small, torch.arange(3, dtype=torch.int32)[None], lengths, dim ** -0.5)


# --------------------------------------------------------- streams and graphs
def _step_inputs(gpu, seed, tokens=3, heads=8, kv=2, dim=128, page=16):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.tensor([31, 200, 64], dtype=torch.int32)
    table, pages = batch(g, lengths.tolist(), page)
    cache = random_cache(g, pages, page, kv, dim)
    row = torch.randn(tokens, heads + 2 * kv, dim, generator=g).bfloat16()
    last = lengths.long() - 1
    slots = table[torch.arange(3), last // page].long() * page + last % page
    cos, sin = angles(256, dim)
    return [t.to(gpu) for t in (row, slots, last, cos, sin, table, lengths)], _to(cache, gpu)


def _step(inputs, cache, heads=8, kv=2):
    row, slots, pos, cos, sin, table, lengths = inputs
    q = qo.kv4_append(cache, row[:, heads:heads + kv], row[:, heads + kv:], slots, positions=pos, cos=cos, sin=sin, q=row[:, :heads])
    return qo.kv4_attention(q, cache, table, lengths)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 60])
def test_positions_next_to_31_bits(gpu, queries, dtype):
    """The longest sequence there may be, over one page, and one that is longer."""
    g = torch.Generator().manual_seed(8)
    cache = random_cache(g, 2, 4096, 1, 64)
    q = torch.randn(queries, 3, 64, generator=g).to(dtype)
    most = 0x7FFFF000
    table = torch.ones(1, most // 4096 + 2, dtype=torch.int32)
    got = _run(gpu, q, cache, table, torch.tensor([most], dtype=torch.int32), window=100)
    check(q, got, cache, torch.ones(1, 1, dtype=torch.int32), torch.tensor([4096], dtype=torch.int32), 0.125, None, 100)
    assert torch.isnan(_run(gpu, q, cache, table, torch.tensor([most + 1], dtype=torch.int32), window=100)).all()


def test_a_step_of_all(gpu):
    """Appended, read and attended to, as a decode step runs them."""
    inputs, cache = _step_inputs(gpu, 1)
    row, slots, pos, cos, sin, table, lengths = (t.cpu() for t in inputs)
    host = tuple(t.cpu().clone() for t in cache)
    got = _step(inputs, cache)
    torch.cuda.synchronize()
    k = ok.turn(row[:, 8:10], pos, cos, sin, False).float()
    for which, x in enumerate((k, row[:, 10:].float())):
        c, s, lo = ok.store(x)
        for t, slot in enumerate(slots.tolist()):
            ok.put(host, which, slot, c[t], s[t], lo[t])
    assert _same([t.cpu() for t in cache], host)
    q = ok.turn(row[:, :8], pos, cos, sin, False).float().bfloat16()
    check(q, got, host, table, lengths, 128 ** -0.5)


def test_on_another_stream(gpu):
    inputs, cache = _step_inputs(gpu, 2)
    want = _step(inputs, _to([t.clone() for t in cache], gpu))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = _step(inputs, cache)
    stream.synchronize()
    assert torch.equal(got, want)


def test_two_graphs_replayed(gpu):
    """Two captured steps, replayed several times in turn with new inputs and eager work between."""
    a, cache_a = _step_inputs(gpu, 3)
    b, cache_b = _step_inputs(gpu, 4)
    long_table = torch.arange(200, dtype=torch.int32, device=gpu)[None]
    long_cache = _to(random_cache(torch.Generator().manual_seed(9), 200, 16, 2, 128), gpu)
    long_n = torch.tensor([3150], dtype=torch.int32, device=gpu)

    def work(inputs, cache):
        return _step(inputs, cache), qo.kv4_attention(inputs[0][:1, :8], long_cache, long_table, long_n)   # shared out, joined

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        for inputs, cache in ((a, cache_a), (b, cache_b)):
            work(inputs, _to([t.clone() for t in cache], gpu))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = work(inputs, cache)
            graphs.append((graph, out, inputs, cache))
    torch.cuda.synchronize()
    for turn in range(4):
        for graph, out, inputs, cache in graphs:
            inputs[0].copy_(torch.randn(inputs[0].shape, generator=torch.Generator().manual_seed(turn)).to(gpu))
            want = work(inputs, _to([t.clone() for t in cache], gpu))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_capi_equals_the_operators(gpu):
    inputs, cache = _step_inputs(gpu, 5)
    row, slots, pos, cos, sin, table, lengths = inputs
    other = _to([t.clone() for t in cache], gpu)
    q = capi.kv4_append(cache, row[:, 8:10], row[:, 10:], slots, pos, cos, sin, row[:, :8])
    assert torch.equal(q, qo.kv4_append(other, row[:, 8:10], row[:, 10:], slots, pos, cos, sin, row[:, :8]))
    assert _same(cache, other)
    for x, y in zip(capi.kv4_read(cache, slots, torch.float16), qo.kv4_read(cache, slots, torch.float16)):
        assert torch.equal(x, y)
    assert torch.equal(capi.kv4_attention(q, cache, table, lengths, 128 ** -0.5, workspace=True),
                       qo.kv4_attention(q, cache, table, lengths))
