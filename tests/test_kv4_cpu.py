"""The 4-bit key/value cache on the host: its formulas against the definition, and what is refused."""
import pytest
import torch

import quant_ops_amd as qo
from kv4_cases import angles, batch, check, random_cache, vectors
from oracle import kv4_reference as ok

DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) or
               (x.dtype == torch.float16 and torch.equal(torch.nan_to_num(x, 7.0), torch.nan_to_num(y, 7.0))) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot,interleaved,page", [(64, 64, False, 16), (96, 48, True, 32), (128, 128, True, 64), (192, 8, False, 16),
                                                      (256, 256, False, 16)])
def test_append_and_read(dim, rot, interleaved, page, dtype):
    g = torch.Generator().manual_seed(dim + rot)
    heads, tokens = 2, 21
    cache = random_cache(g, 4, page, heads, dim)
    want = tuple(t.clone() for t in cache)
    row = vectors(g, tokens, 3 + 2 * heads, dim).to(dtype)
    q, k, v = row[:, :3], row[:, 3:5], row[:, 5:]
    slots = torch.randperm(4 * page, generator=g)[:tokens]
    slots[3], slots[7] = -1, 4 * page
    pos = torch.randint(0, 50, (tokens,), generator=g)
    cos, sin = angles(50, rot)
    got = qo.kv4_append(cache, k, v, slots, positions=pos, cos=cos, sin=sin, q=q, interleaved=interleaved)
    assert torch.equal(got, ok.turn(q, pos, cos, sin, interleaved).float().to(dtype))
    for which, x in enumerate((ok.turn(k, pos, cos, sin, interleaved).float(), v.float())):
        c, s, lo = ok.store(x)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < 4 * page:
                ok.put(want, which, slot, c[t], s[t], lo[t])
    assert _same(cache, want)
    for out_dtype in DTYPES:
        for which, x in enumerate(qo.kv4_read(cache, slots, out_dtype)):
            assert x.dtype == out_dtype
            for t, slot in enumerate(slots.tolist()):
                row = ok.read(want, which, slot, out_dtype) if 0 <= slot < 4 * page else torch.zeros(heads, dim, dtype=out_dtype)
                assert torch.equal(x[t], row)


def test_vectors_at_the_edges():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(9, 1, 64, generator=g)
    x[0] = 3.25                                     # constant
    x[1] = 0.0
    x[2, 0, 5], x[3, 0, 63], x[4, 0, 0] = float("nan"), float("inf"), -float("inf")
    x[5] *= 1e30                                    # past fp16
    x[6] *= 1e-30                                   # below it
    x[7] = torch.arange(64) * 0.5 / 2 - 3           # ties between codes
    x[8] = 1000 + 0.001 * x[8]
    cache = qo.kv4_cache(1, 16, 1, 64, device="cpu")
    qo.kv4_append(cache, x, -x, torch.arange(9))
    for which, v in enumerate((x, -x)):
        c, s, lo = ok.store(v)
        want = tuple(t.clone() for t in cache)
        for t in range(9):
            ok.put(want, which, t, c[t], s[t], lo[t])
        assert _same(cache, want)
    k, v = qo.kv4_read(cache, torch.arange(9))
    assert torch.equal(torch.isnan(k).all(2)[:, 0], torch.tensor([0, 0, 1, 1, 1, 0, 0, 0, 0]).bool())
    assert torch.equal(k[0], x[0]) and torch.equal(k[1], x[1])
    # 15 steps of fp16(131008 / 15) from -65504: past fp16's largest by half a step
    assert k[5].max() == 65536 and qo.kv4_read(cache, torch.tensor([5]), torch.float16)[0].max() == 65504


def test_position_outside_the_table():
    cache = qo.kv4_cache(1, 16, 1, 64, device="cpu")
    cos, sin = angles(4, 32)
    x = torch.ones(3, 1, 64)
    got = qo.kv4_append(cache, x, x, torch.arange(3), positions=torch.tensor([1, 4, -1]), cos=cos, sin=sin, q=x)
    assert torch.isnan(got[1:, :, :32]).all() and not torch.isnan(got[0]).any() and not torch.isnan(got[:, :, 32:]).any()
    k, v = qo.kv4_read(cache, torch.arange(3))
    assert torch.isnan(k[1:]).all() and not torch.isnan(k[0]).any() and not torch.isnan(v).any()


CASES = [   # lengths, query heads, KV heads, head_dim, page, queries each (a list: ragged, with two rows behind), window
    ([1, 15, 16, 17, 64, 65, 130, 0], 4, 2, 64, 16, 1, 0),
    ([40, 3, 70], 3, 3, 96, 32, 5, 0),
    ([50, 1, 0, 33], 8, 1, 128, 16, [7, 1, 2, 0], 0),
    ([90, 20], 6, 2, 192, 64, 3, 17),
    ([100, 64, 5], 2, 1, 256, 16, [30, 0, 5], 1),
]


def make(case, dtype, seed=0):
    lengths, heads, kv, dim, page, queries, window = case
    g = torch.Generator().manual_seed(seed + sum(lengths) + dim)
    table, pages = batch(g, lengths, page)
    cache = random_cache(g, pages, page, kv, dim)
    starts = None
    rows = queries * len(lengths) if isinstance(queries, int) else sum(queries) + 2
    if not isinstance(queries, int):
        starts = torch.tensor([sum(queries[:i]) for i in range(len(queries) + 1)], dtype=torch.int32)
    q = (1.5 * torch.randn(rows, heads, dim, generator=g)).to(dtype)
    return q, cache, table, torch.tensor(lengths, dtype=torch.int32), starts, window


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_attention(case, dtype):
    q, cache, table, lengths, starts, window = make(case, dtype)
    got = qo.kv4_attention(q, cache, table, lengths, q_starts=starts, window=window)
    assert got.dtype == dtype and got.shape == q.shape
    check(q, got, cache, table, lengths, q.shape[2] ** -0.5, starts, window)


def test_masked_places_may_hold_anything():
    """NaN behind the last token, in tokens before the window, and in a token that only later queries see."""
    q, cache, table, lengths, _, _ = make(([37], 2, 1, 64, 16, 4, 10), torch.float32)
    flat = cache.params
    for t in list(range(37, 48)) + list(range(0, 24)) + [35]:   # the queries stand at 33 .. 36 and see from 24 on
        page, place = int(table[0, t // 16]), t % 16
        flat[page, :, :, place // 16, :, place % 16] = float("nan")
    got = qo.kv4_attention(q, cache, table, lengths, window=10)
    assert not torch.isnan(got[:2]).any() and torch.isnan(got[2:]).all()
    check(q, got, cache, table, lengths, 64 ** -0.5, None, 10)


def test_bad_pages_and_lengths():
    q, cache, table, lengths, _, _ = make(([40, 40, 40, 40, -3], 2, 1, 64, 16, 1, 0), torch.float32)
    table[0, 1], table[1, 2], lengths[2] = -1, cache.k_codes.shape[0], 16 * table.shape[1] + 1
    got = qo.kv4_attention(q, cache, table, lengths)
    assert [bool(torch.isnan(got[i]).all()) for i in range(5)] == [True, True, True, False, False]
    assert not torch.isnan(got[3:]).any() and not got[4].any()
    check(q, got, cache, table, lengths, 64 ** -0.5)


def refusals(device):
    """Calls that are refused, on tensors of the device."""
    cache = qo.kv4_cache(2, 16, 2, 64, device=device)
    x = torch.zeros(3, 2, 64, device=device)
    slots, pos = torch.arange(3, device=device), torch.arange(3, device=device)
    cos = torch.ones(4, 32, device=device)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32, device=device), torch.ones(3, dtype=torch.int32, device=device)
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=device)
    other = qo.KV4Cache(cache.k_codes, cache.v_codes[:1], cache.params)
    strided = qo.KV4Cache(cache.k_codes.transpose(0, 1).contiguous().transpose(0, 1), cache.v_codes, cache.params)
    odd = [qo.KV4Cache(torch.zeros(2, 1, p, d // 2, dtype=torch.uint8, device=device),
                       torch.zeros(2, 1, p // 16, d // 2, 16, dtype=torch.uint8, device=device),
                       torch.zeros(2, 2, 1, p // 16, 2, 16, dtype=torch.float16, device=device)) for p, d in ((48, 64), (16, 80), (16, 320), (8192, 64))]
    turn = dict(positions=pos, cos=cos, sin=cos)
    headless = qo.KV4Cache(cache.k_codes[:, :0].contiguous(), cache.v_codes[:, :0].contiguous(), cache.params[:, :, :0].contiguous())
    return [
        lambda: qo.kv4_append(cache, x.double(), x.double(), slots),
        lambda: qo.kv4_append(cache, x, x.half(), slots),
        lambda: qo.kv4_append(cache, x[:, :1], x[:, :1], slots),
        lambda: qo.kv4_append(cache, x[..., :32], x[..., :32], slots),
        lambda: qo.kv4_append(cache, x, x[:2], slots),
        lambda: qo.kv4_append(cache, x[0], x[0], slots),
        lambda: qo.kv4_append(cache, x, x, slots[:2]),
        lambda: qo.kv4_append(cache, x, x, slots.int()),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos),
        lambda: qo.kv4_append(cache, x, x, slots, cos=cos, sin=cos),
        lambda: qo.kv4_append(cache, x, x, slots, q=x),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos.int(), cos=cos, sin=cos),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos[:2], cos=cos, sin=cos),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos, cos=cos.half(), sin=cos.half()),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos, cos=cos, sin=cos[:2]),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos, cos=cos[:0], sin=cos[:0]),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos, cos=cos[:, :6], sin=cos[:, :6]),
        lambda: qo.kv4_append(cache, x, x, slots, positions=pos, cos=torch.cat((cos, cos), 1), sin=torch.cat((cos, cos), 1)),
        lambda: qo.kv4_append(cache, x, x, slots, q=x.half(), **turn),
        lambda: qo.kv4_append(cache, x, x, slots, q=x[:2], **turn),
        lambda: qo.kv4_append(other, x, x, slots),
        lambda: qo.kv4_append(strided, x, x, slots),
        lambda: qo.kv4_append(qo.KV4Cache(cache.k_codes.int(), cache.v_codes, cache.params), x, x, slots),
        lambda: qo.kv4_append(qo.KV4Cache(cache.k_codes, cache.v_codes, cache.params.float()), x, x, slots),
        lambda: qo.kv4_append(odd[0], x[:, :1], x[:, :1], slots),
        lambda: qo.kv4_read(odd[1], slots),
        lambda: qo.kv4_read(odd[2], slots),
        lambda: qo.kv4_read(odd[3], slots),
        lambda: qo.kv4_read(cache, slots.int()),
        lambda: qo.kv4_read(cache, slots[None]),
        lambda: qo.kv4_read(cache, slots, out_dtype=torch.float64),
        lambda: qo.kv4_read(cache, slots, out_dtype=torch.uint8),
        lambda: qo.kv4_attention(x.double(), cache, table, lengths),
        lambda: qo.kv4_attention(x[0], cache, table, lengths),
        lambda: qo.kv4_attention(x[..., :32], cache, table, lengths),
        lambda: qo.kv4_attention(x[:, :1], cache, table, lengths),
        lambda: qo.kv4_attention(x[:, :0], cache, table, lengths),
        lambda: qo.kv4_attention(x, cache, table.long(), lengths),
        lambda: qo.kv4_attention(x, cache, table[0], lengths),
        lambda: qo.kv4_attention(x, cache, table, lengths.long()),
        lambda: qo.kv4_attention(x, cache, table, lengths[:2]),
        lambda: qo.kv4_attention(x, cache, table[:2], lengths[:2]),
        lambda: qo.kv4_attention(x, cache, table[:0], lengths[:0]),
        lambda: qo.kv4_attention(x, cache, table, lengths, q_starts=starts[:3]),
        lambda: qo.kv4_attention(x, cache, table, lengths, q_starts=starts.long()),
        lambda: qo.kv4_attention(x, cache, table, lengths, scale=0.0),
        lambda: qo.kv4_attention(x, cache, table, lengths, scale=-1.0),
        lambda: qo.kv4_attention(x, cache, table, lengths, scale=float("nan")),
        lambda: qo.kv4_attention(x, cache, table, lengths, scale=float("inf")),
        lambda: qo.kv4_attention(x, cache, table, lengths, window=-1),
        lambda: qo.kv4_attention(x, other, table, lengths),
        lambda: qo.kv4_attention(x, odd[1], table, lengths),
        lambda: qo.kv4_attention(x, headless, table, lengths),
        lambda: qo.kv4_append(headless, x[:, :0], x[:, :0], slots),
        lambda: qo.kv4_read(headless, slots),
    ]


def check_refused(calls):
    for i, call in enumerate(calls):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was accepted")


def test_refusals():
    check_refused(refusals("cpu"))
    for size in ((2, 48, 1, 64), (2, 16, 1, 100), (2, 8, 1, 64), (-1, 16, 1, 64), (2, 16, 0, 64), (2, 8192, 1, 64)):
        with pytest.raises(ValueError):
            qo.kv4_cache(*size, device="cpu")


def test_fakes():
    """Shapes and types under tracing."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    if not qo.CUDA_AVAILABLE:
        pytest.skip("library not built")
    with FakeTensorMode():
        cache = qo.kv4_cache(2, 16, 2, 64)
        x = torch.empty(3, 4, 64, device="cuda", dtype=torch.bfloat16)
        slots = torch.empty(3, dtype=torch.int64, device="cuda")
        cos = torch.empty(8, 32, device="cuda")
        got = qo.kv4_append(cache, x[:, :2], x[:, 2:], slots, positions=slots, cos=cos, sin=cos, q=x)
        assert got.shape == x.shape and got.dtype == x.dtype
        assert qo.kv4_append(cache, x[:, :2], x[:, 2:], slots) is None
        k, v = qo.kv4_read(cache, slots, torch.float16)
        assert k.shape == v.shape == (3, 2, 64) and k.dtype == torch.float16
        table, n = torch.empty(3, 2, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
        assert qo.kv4_attention(x, cache, table, n).shape == x.shape
