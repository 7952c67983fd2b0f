"""The operators of a key/value cache held in 4 bits as timed and checked cases: appending keys and values with the
position rotation, reading them back, and attention over the cache.

Format: per token and KV head one vector v of D values. v is clamped to +-65504; lo = fp16(min v), s = fp16((max v -
lo) / 15), c = (v - lo) / s rounded to nearest even and clamped to 0 .. 15 (s = 0: 0); the vector reads as lo + s c.
Pages of P tokens (slot = page * P + place), laid out as

    k_codes uint8   [pages, Hkv, P, D / 2]           byte j: value 2j in the low bits, 2j + 1 in the high
    v_codes uint8   [pages, Hkv, P / 16, D / 2, 16]  the same bytes, 16 tokens side by side
    params  float16 [pages, 2, Hkv, P / 16, 2, 16]   keys, values; s, lo; 16 tokens side by side

Rotation of the first R values of a vector by its position's angles (float32 tables [positions, R / 2]): pairs
(i, i + R / 2), or (2i, 2i + 1) where interleaved; the rotated values are rounded to float32, then quantized.

Attention: query i of n of a sequence of L tokens stands at p = L - n + i and sees the tokens up to p (of a
window: the last `window` of them). Nothing to see gives 0.

Sizes are generic; batches run from one decoded token to a prefill of 8192, contexts to 131072 tokens.
"""
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
HEAD_DIMS = (64, 96, 128, 192, 256)
PAGES = (16, 32, 64, 128, 256)
GROUPS = (1, 2, 3, 4, 5, 6, 7, 8, 16)

# The largest listed work, which bounds the drawn cases.
MOST_MOVED = 8192 * (32 + 2 * 8) * 128   # values of an append's or a read's tokens
MOST_CACHED = 131072 * 8 * 128           # values of an attention's keys
MOST_SCORES = 2048 * 4096 * 32           # (query, head, token) triples


def listed():
    return [
        # one decoded token's queries, keys and values
        {"name": "append_bf16_1x32x8x128", "kind": "append", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "page": 64, "dtype": "bf16"},
        # a large decode batch, half of each head rotated in interleaved pairs
        {"name": "append_fp16_257x16x16x64", "kind": "append", "tokens": 257, "heads": 16, "kv_heads": 16, "dim": 64,
         "rot": 32, "interleaved": True, "page": 16, "dtype": "fp16"},
        # a large prefill
        {"name": "append_bf16_8192x32x8x128", "kind": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "page": 64, "dtype": "bf16"},
        # a short shared prefix read back
        {"name": "read_fp32_333x4x96", "kind": "read", "tokens": 333, "kv_heads": 4, "dim": 96, "page": 16,
         "dtype": "fp32"},
        # a long one
        {"name": "read_bf16_8192x8x128", "kind": "read", "tokens": 8192, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16"},
        # one user's next token, early in a chat
        {"name": "decode_bf16_1x32x8x128_700", "kind": "attention", "batch": 1, "queries": 1, "ragged": False,
         "longest": 700, "shortest": 700, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0,
         "dtype": "bf16"},
        # a busy server's decode step: contexts of all lengths
        {"name": "decode_bf16_64x32x8x128_4096", "kind": "attention", "batch": 64, "queries": 1, "ragged": False,
         "longest": 4096, "shortest": 100, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0,
         "dtype": "bf16"},
        # every query head with keys of its own, small pages
        {"name": "decode_fp16_16x32x32x128_2048", "kind": "attention", "batch": 16, "queries": 1, "ragged": False,
         "longest": 2048, "shortest": 1, "heads": 32, "kv_heads": 32, "dim": 128, "page": 16, "window": 0,
         "dtype": "fp16"},
        # one very long document
        {"name": "decode_bf16_1x64x8x128_131072", "kind": "attention", "batch": 1, "queries": 1, "ragged": False,
         "longest": 131072, "shortest": 131072, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "window": 0,
         "dtype": "bf16"},
        # four proposed tokens of each sequence checked at once, float32, wide heads, a sliding window
        {"name": "verify_fp32_24x16x8x256_w1024", "kind": "attention", "batch": 24, "queries": 4, "ragged": False,
         "longest": 3000, "shortest": 2, "heads": 16, "kv_heads": 8, "dim": 256, "page": 32, "window": 1024,
         "dtype": "fp32"},
        # chunks of prompts beside decoded tokens in one ragged batch, with rows of padding behind
        {"name": "mixed_fp16_8x24x4x64_2000", "kind": "attention", "batch": 8, "queries": 500, "ragged": True,
         "longest": 2000, "shortest": 300, "heads": 24, "kv_heads": 4, "dim": 64, "page": 16, "window": 0,
         "dtype": "fp16"},
        # the second chunk of a long prompt
        {"name": "prefill_bf16_2048x32x8x128_4096", "kind": "attention", "batch": 1, "queries": 2048, "ragged": False,
         "longest": 4096, "shortest": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choices(("append", "read", "attention"), (3, 2, 6))[0]
    dim, page = rng.choice(HEAD_DIMS), rng.choice(PAGES)
    dtype = rng.choices(("bf16", "fp16", "fp32"), (5, 3, 2))[0]
    kv_heads = _log(rng, 1, 32)
    if kind == "read":
        return {"kind": kind, "tokens": _log(rng, 1, min(8192, MOST_MOVED // (2 * kv_heads * dim))),
                "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    group = rng.choice([g for g in GROUPS if g * kv_heads <= 128])
    if kind == "append":
        heads = group * kv_heads
        return {"kind": kind, "tokens": _log(rng, 1, min(8192, MOST_MOVED // ((heads + 2 * kv_heads) * dim))),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rng.choice((dim, dim, dim // 2)),
                "interleaved": rng.random() < 0.4, "page": page, "dtype": dtype}
    ragged = rng.random() < 0.3
    batch = _log(rng, 1, 16 if ragged else 128)
    longest = _log(rng, 1, MOST_CACHED // (batch * kv_heads * dim))
    longest = min(longest, 131072, max(1, MOST_SCORES // (batch * group * kv_heads)))
    room = min(2048, longest, max(1, MOST_SCORES // (batch * group * kv_heads * longest)))
    queries = _log(rng, 1, room) if ragged or rng.random() < 0.4 else 1
    return {"kind": kind, "batch": batch, "queries": queries, "ragged": ragged, "longest": longest,
            "shortest": max(queries, longest // rng.choice((1, 2, 10, 1000))), "heads": group * kv_heads,
            "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": _log(rng, 1, 8192) if rng.random() < 0.2 else 0, "dtype": dtype}


def _lengths(case):
    """Tokens and queries of each sequence, longest first."""
    b, most, least, n = case["batch"], case["longest"], case["shortest"], case["queries"]
    tokens = [most - (most - least) * i // max(1, b - 1) for i in range(b)]
    if not case["ragged"]:
        return tokens, [n] * b
    return tokens, [1 if i % 2 else min(t, max(1, n * (b - i) // b)) for i, t in enumerate(tokens)]


TAIL = 5   # rows behind the last sequence of a ragged batch


# ----------------------------------------------------------------- plain forms
def _split(v):
    """Codes [..., D] (uint8), s and lo [...] (float16) of float32 vectors."""
    v = v.clamp(-65504, 65504)
    lo = v.amin(-1).half()
    s = ((v.amax(-1).double() - lo.double()) / 15).clamp(min=0).half()
    # borders between codes: in 64 bits
    c = (v.double() - lo.double()[..., None]) / torch.where(s == 0, 1.0, s.double())[..., None]
    return torch.where(s[..., None] == 0, 0.0, torch.round(c).clamp(0, 15)).to(torch.uint8), s, lo


def _rotate(x, cos, sin, rot, interleaved):
    """x [T, H, D] with its first `rot` values rotated by the angles of cos, sin [T, rot / 2]: float32."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]   # each value decides between two codes
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack((a, b), 3).flatten(2) if interleaved else torch.cat((a, b), 2)
    return torch.cat((turned, x[..., rot:]), 2).float()


def _round_trip(v):
    """What a vector reads as: float32."""
    c, s, lo = _split(v)
    return lo.float()[..., None] + s.float()[..., None] * c.float()


def _cached(s, page, place):
    """float32 keys and values [..., Hkv, D] at (page, place)."""
    def values(codes, which):
        nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
        par = s["params"][page, which, :, place // 16, :, place % 16].float()   # [..., Hkv, 2]
        return par[..., 1:] + par[..., :1] * nib

    return (values(s["k_codes"][page, :, place], 0),
            values(s["v_codes"][page, :, place // 16, :, place % 16], 1))


def _attend(s):
    case = s["case"]
    b, heads, kv, dim, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    g, n, most = heads // kv, case["queries"], case["longest"]
    t = torch.arange(most, device="cuda")
    at = s["table"].long().clamp(min=0)[:, t // page]
    k, v = _cached(s, at, (t % page).expand(b, most))                  # [b, most, kv, dim]
    k = k.permute(0, 2, 3, 1).reshape(b * kv, dim, most).contiguous()
    v = v.permute(0, 2, 1, 3).reshape(b * kv, most, dim).contiguous()
    lengths = s["lengths"].long()
    if case["ragged"]:
        starts = s["q_starts"].long()
        counts = starts[1:] - starts[:-1]
    else:
        starts = torch.arange(b + 1, device="cuda") * n
        counts = torch.full((b,), n, device="cuda")
    i = torch.arange(n, device="cuda")
    there = i < counts[:, None]                                        # [b, n]
    rows = torch.where(there, starts[:-1, None] + i, 0)
    q = s["q"].float()[rows].view(b, n, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(b * kv, n * g, dim).contiguous()
    score = torch.bmm(q, k).view(b, kv, n, g, most).mul_(s["scale"])
    pos = (lengths - counts)[:, None] + i
    seen = (t <= pos[..., None]) & there[..., None]
    if case["window"]:
        seen &= t > pos[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = score.amax(4, keepdim=True)
    p = score.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(4, keepdim=True)
    o = torch.bmm(p.view(b * kv, n * g, most), v).view(b, kv, n, g, dim) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, heads, dim)
    out = torch.zeros_like(s["q"])
    out[rows[there]] = o[there].to(out.dtype)
    return out


# ----------------------------------------------------------------------- cases
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys(g, *shape):
    """N(0, 1), the same few channels of each head larger, as rotated keys have them."""
    x = torch.randn(*shape, generator=g, device="cuda")
    x[..., torch.randperm(shape[-1], generator=g, device="cuda")[: shape[-1] // 32]] *= 4.0
    return x


def _fill(s, g, pages, case):
    """A cache that holds keys and values already, as earlier steps left it."""
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    for which in ("k", "v"):
        x = _keys(g, pages, kv, page, dim) if which == "k" else torch.randn(pages, kv, page, dim, generator=g, device="cuda")
        c, scale, lo = _split(x)
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
        if which == "v":
            codes = codes.view(pages, kv, page // 16, 16, dim // 2).transpose(3, 4).contiguous()
        s[which + "_codes"] = codes
        s[which] = torch.stack((scale.view(pages, kv, page // 16, 16), lo.view(pages, kv, page // 16, 16)), 3)
    s["params"] = torch.stack((s.pop("k"), s.pop("v")), 1)


def _slots(g, case):
    """Slots of a few sequences' tokens in pages all over the cache, and its number of pages."""
    tokens, page = case["tokens"], case["page"]
    pages = -(-tokens // page) * 2 + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    t = torch.arange(tokens, device="cuda") + int(torch.randint(0, page, (1,), generator=g, device="cuda"))
    return order[t // page] * page + t % page, pages


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    kv, dim, page, dtype = case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    if kind == "append":
        tokens, heads, rot = case["tokens"], case["heads"], case["rot"]
        s["slots"], pages = _slots(g, case)
        s["k_codes"] = torch.zeros(pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
        s["v_codes"] = torch.zeros(pages, kv, page // 16, dim // 2, 16, dtype=torch.uint8, device="cuda")
        s["params"] = torch.zeros(pages, 2, kv, page // 16, 2, 16, dtype=torch.float16, device="cuda")
        # queries, keys and values as the projection gives them: side by side in one row
        row = _keys(g, tokens, heads + 2 * kv, dim).to(dtype)
        s["q"], s["k"], s["v"] = row[:, :heads], row[:, heads:heads + kv], row[:, heads + kv:]
        angle = torch.arange(16384, device="cuda").double()[:, None] * 10000.0 ** (
            -torch.arange(0, rot, 2, device="cuda").double() / rot)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = torch.arange(tokens, device="cuda") + int(torch.randint(0, 8000, (1,), generator=g, device="cuda"))
    elif kind == "read":
        s["slots"], pages = _slots(g, case)
        _fill(s, g, pages, case)
    else:
        b, heads = case["batch"], case["heads"]
        lengths, counts = _lengths(case)
        order = torch.randperm(b, generator=g, device="cuda").tolist()
        lengths, counts = [lengths[i] for i in order], [counts[i] for i in order]
        need = [-(-n // page) for n in lengths]
        _fill(s, g, sum(need) + 2, case)
        ids = torch.randperm(sum(need) + 2, generator=g, device="cuda").to(torch.int32).cpu()
        table = torch.full((b, -(-case["longest"] // page)), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = ids[at:at + n]
            at += n
        s["table"] = table.cuda()
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q_starts"] = None
        if case["ragged"]:
            s["q_starts"] = torch.tensor([sum(counts[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
        rows = sum(counts) + (TAIL if case["ragged"] else 0)
        s["q"] = (1.5 * torch.randn(rows, heads, dim, generator=g, device="cuda")).to(dtype)
        s["scale"] = dim ** -0.5
    return s


def _run_own(s):
    import quant_ops_amd as qo

    case = s["case"]
    cache = qo.KV4Cache(s["k_codes"], s["v_codes"], s["params"])
    if case["kind"] == "append":
        q = qo.kv4_append(cache, s["k"], s["v"], s["slots"], positions=s["positions"], cos=s["cos"], sin=s["sin"],
                          q=s["q"], interleaved=case["interleaved"])
        return (q, *qo.kv4_read(cache, s["slots"], out_dtype=s["k"].dtype))
    if case["kind"] == "read":
        return qo.kv4_read(cache, s["slots"], out_dtype=DTYPES[case["dtype"]])
    return qo.kv4_attention(s["q"], cache, s["table"], s["lengths"], scale=s["scale"], q_starts=s["q_starts"],
                            window=case["window"])


def run(s):
    """One pass. Appended vectors come back as the values that they read as."""
    if own:
        return _run_own(s)
    case = s["case"]
    if case["kind"] == "append":
        c, d, rot = s["cos"][s["positions"]], s["sin"][s["positions"]], case["rot"]
        dtype = s["k"].dtype
        return (_rotate(s["q"], c, d, rot, case["interleaved"]).to(dtype),
                _round_trip(_rotate(s["k"], c, d, rot, case["interleaved"])).to(dtype),
                _round_trip(s["v"].float()).to(dtype))
    if case["kind"] == "read":
        k, v = _cached(s, s["slots"] // case["page"], s["slots"] % case["page"])
        return k.to(DTYPES[case["dtype"]]), v.to(DTYPES[case["dtype"]])
    return _attend(s)


def work(case):
    kv, dim, es = case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    vector = dim // 2 + 4   # bytes of a vector in the cache
    if case["kind"] == "append":
        t, h = case["tokens"], case["heads"]
        # read and written: q; read: k, v and the angles; written and read back: the cache; written: k and v again
        return {"bytes": t * (2 * h * dim * es + 2 * kv * dim * es + case["rot"] * 4 + 2 * 2 * kv * vector + 2 * kv * dim * es),
                "flops": t * (3 * (h + kv) * case["rot"] + 2 * 8 * kv * dim)}
    if case["kind"] == "read":
        return {"bytes": case["tokens"] * kv * 2 * (vector + dim * es), "flops": case["tokens"] * kv * 2 * 2 * dim}
    pairs = cached = rows = 0
    for length, n in zip(*_lengths(case)):
        w = case["window"] or length
        # sum over the queries' positions p of min(p + 1, w)
        first, last = max(0, length - n) + 1, length
        full = max(0, last - max(first, w) + 1)
        ramp = max(0, min(last, w - 1) - first + 1)
        pairs += full * w + ramp * (2 * first + ramp - 1) // 2
        cached += min(length, w + n - 1)
        rows += n
    return {"bytes": 2 * rows * case["heads"] * dim * es + cached * kv * 2 * vector,
            "flops": 4 * dim * case["heads"] * pairs}


# -------------------------------------------------------- the definition in 64 bits
def _exact_turn(x, angles, rot, interleaved):
    """Rotation as the product with 2 x 2 matrices."""
    c, s = (a.double() for a in angles)
    mat = torch.stack((torch.stack((c, -s), -1), torch.stack((s, c), -1)), -2)          # [T, R / 2, 2, 2]
    head = x[..., :rot].double()
    pairs = (head.reshape(*x.shape[:2], rot // 2, 2) if interleaved else
             head.reshape(*x.shape[:2], 2, rot // 2).transpose(2, 3))
    pairs = (mat[:, None] * pairs[..., None, :]).sum(-1)
    out = x.double().clone()
    out[..., :rot] = (pairs if interleaved else pairs.transpose(2, 3)).reshape(*x.shape[:2], rot)
    return out


def _exact_store(x):
    """The value nearest to each of a vector's among lo + s c, c = 0 .. 15 (the even c of two); the vector
    itself, lo and s are rounded as the format says."""
    x = x.float().double().clamp(-65504, 65504)
    lo = x.min(-1, keepdim=True).values.half().double()
    s = ((x.max(-1, keepdim=True).values - lo) / 15).clamp(min=0).half().double()
    below = torch.where(s > 0, torch.floor((x - lo) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15)
    left, right = x - (lo + s * below), (lo + s * (below + 1)) - x
    up = (right < left) | ((right == left) & (below % 2 == 1))
    return lo + s * torch.where(up & (below < 15) & (s > 0), below + 1, below)


def _exact_rows(s, page, place):
    """Keys and values [..., Hkv, D] in 64 bits at (page, place)."""
    got = []
    for which, codes in enumerate((s["k_codes"][page, :, place], s["v_codes"][page, :, place // 16, :, place % 16])):
        whole = codes.to(torch.int64)
        nib = torch.empty(*whole.shape[:-1], 2 * whole.shape[-1], dtype=torch.float64, device=whole.device)
        nib[..., 0::2], nib[..., 1::2] = (whole % 16).double(), (whole // 16).double()
        scale = s["params"][page, which, :, place // 16, 0, place % 16].double()
        least = s["params"][page, which, :, place // 16, 1, place % 16].double()
        got.append(nib * scale[..., None] + least[..., None])
    return got


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "append":
        angles = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return (_exact_turn(s["q"], angles, case["rot"], case["interleaved"]),
                _exact_store(_exact_turn(s["k"], angles, case["rot"], case["interleaved"])),
                _exact_store(s["v"].double()))
    if kind == "read":
        return tuple(_exact_rows(s, s["slots"] // case["page"], s["slots"] % case["page"]))
    heads, kv, page = case["heads"], case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lengths = s["lengths"].tolist()
    n = case["queries"]
    starts = s["q_starts"].tolist() if case["ragged"] else [n * i for i in range(case["batch"] + 1)]
    for b, length in enumerate(lengths):
        t = torch.arange(length, device="cuda")
        k, v = _exact_rows(s, s["table"][b].long()[t // page], t % page)     # [length, kv, dim]
        q = s["q"][starts[b]:starts[b + 1]].double()
        pos = torch.arange(length - len(q), length, device="cuda")[:, None]
        hidden = (t > pos) | ((t <= pos - case["window"]) if case["window"] else torch.zeros_like(t > pos))
        for h in range(heads):
            score = (q[:, h] * s["scale"]) @ k[:, h // (heads // kv)].t().contiguous()
            p = torch.softmax(score.masked_fill(hidden, float("-inf")), 1).masked_fill(hidden, 0.0)   # no token: 0
            out[starts[b]:starts[b + 1], h] = p @ v[:, h // (heads // kv)].contiguous()
    return out
