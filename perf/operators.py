"""The microscaled (MX) operators as timed and checked cases: quantizing to 4 and 8 bits, the RMS norm with the
residual's addition and the SwiGLU gate that quantize their result, the product with 4-bit weights, and the MLP
block that runs them together.

MX formats: 32 consecutive values of a row share a scale 2^e, held as the byte e + 127; the codes are FP4 e2m1 (two
per byte, the even value in the low bits) or FP8 e4m3. Rows that are no whole number of blocks are padded with
zeros. Widths and projections are those of this repository's tests and benchmark, or generic; token counts run from
one decoded token to a prefill of 8192.
"""
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6

# hidden and FFN widths of the repository's tests
WIDTHS = (1024, 1536, 2048, 2560, 3584, 4096, 5120, 5632, 6144, 6912, 7168, 8192, 8960, 9216, 9728, 10240, 11008,
          12288, 13696, 13824, 14336, 16384, 18432, 18944, 20480, 22016, 24576, 25600, 27648, 28672)

# (out, in) features of projections over those widths
PROJECTIONS = ((4096, 4096), (6144, 4096), (14336, 4096), (4096, 14336), (11008, 4096), (4096, 11008), (5120, 5120),
               (13824, 5120), (5120, 13824), (3584, 3584), (18944, 3584), (3584, 18944), (8192, 8192), (28672, 8192),
               (8192, 28672), (1024, 4096), (2048, 2048))

# (hidden, FFN) widths of MLP blocks over those projections
BLOCKS = ((4096, 14336), (4096, 11008), (3584, 18944), (5120, 13824), (2048, 5632), (1024, 2560))

# The largest listed work, which bounds the drawn cases.
MOST_ELEMENTS = 14336 * 4096
MOST_PRODUCTS = 4096 * 14336 * 4096


def listed():
    return [
        # a decode batch's activations before a product with 4-bit weights
        {"name": "quantize_fp4_bf16_16x14336", "kind": "quantize", "tokens": 16, "features": 14336, "dtype": "bf16",
         "fmt": "fp4"},
        # loading a weight: a gate projection rounded to 4 bits
        {"name": "quantize_fp4_bf16_14336x4096", "kind": "quantize", "tokens": 14336, "features": 4096, "dtype": "bf16",
         "fmt": "fp4"},
        # a ragged batch of rows that end inside a block, in 8 bits
        {"name": "quantize_fp8_fp16_1021x5000", "kind": "quantize", "tokens": 1021, "features": 5000, "dtype": "fp16",
         "fmt": "fp8"},
        # one decoded token: what the previous layer gave, added to the residual stream and normed
        {"name": "norm_fp8_bf16_1x4096", "kind": "norm", "tokens": 1, "features": 4096, "dtype": "bf16",
         "residual": True, "fmt": "fp8"},
        # the same before an MLP in a large prefill
        {"name": "norm_fp8_bf16_8192x4096", "kind": "norm", "tokens": 8192, "features": 4096, "dtype": "bf16",
         "residual": True, "fmt": "fp8"},
        # the gate of a decode batch
        {"name": "swiglu_fp8_bf16_16x14336", "kind": "swiglu", "tokens": 16, "features": 14336, "dtype": "bf16",
         "fmt": "fp8"},
        # the gate of a prefill, fp16
        {"name": "swiglu_fp8_fp16_2048x14336", "kind": "swiglu", "tokens": 2048, "features": 14336, "dtype": "fp16",
         "fmt": "fp8"},
        # one decoded token through the down projection, 8-bit activations
        {"name": "matmul_fp8_1x4096x14336", "kind": "matmul", "m": 1, "n": 4096, "k": 14336, "fmt": "fp8", "bias": False,
         "out": "bf16"},
        # a mixed decode / prefill batch against a smaller FFN's gate projection, with bias
        {"name": "matmul_fp8_333x11008x4096", "kind": "matmul", "m": 333, "n": 11008, "k": 4096, "fmt": "fp8",
         "bias": True, "out": "bf16"},
        # the gate projection of a prefill, 4-bit activations
        {"name": "matmul_fp4_4096x14336x4096", "kind": "matmul", "m": 4096, "n": 14336, "k": 4096, "fmt": "fp4",
         "bias": False, "out": "bf16"},
        # a whole MLP block for a decode batch, 8-bit activations
        {"name": "mlp_fp8_16x4096x14336", "kind": "mlp", "tokens": 16, "hidden": 4096, "ffn": 14336, "fmt": "fp8"},
        # and for one chunk of a chunked prefill, 4-bit activations
        {"name": "mlp_fp4_1024x4096x14336", "kind": "mlp", "tokens": 1024, "hidden": 4096, "ffn": 14336, "fmt": "fp4"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng):
    """A width of the tests, or any other: rows that end inside a block, or inside a 16-byte piece, among them."""
    return rng.choice(WIDTHS) if rng.random() < 0.6 else _log(rng, 100, 28672)


def draw(rng):
    kind = rng.choices(("quantize", "norm", "swiglu", "matmul", "mlp"), (4, 4, 3, 7, 2))[0]
    if kind in ("quantize", "norm", "swiglu"):
        features = _width(rng)
        most = MOST_ELEMENTS // features // (2 if kind == "swiglu" else 1)
        case = {"kind": kind, "tokens": _log(rng, 1, min(8192, most)), "features": features,
                "dtype": rng.choices(("bf16", "fp16", "fp32"), (5, 3, 2))[0],
                "fmt": rng.choice(("fp4", "fp8")) if kind == "quantize" else "fp8"}
        if kind == "norm":
            case["residual"] = rng.random() < 0.7
        return case
    if kind == "matmul":
        n, k = rng.choice(PROJECTIONS)
        if rng.random() < 0.3:   # any out width, any whole number of blocks
            n, k = _log(rng, 200, 16384), 32 * _log(rng, 16, 448)
        return {"kind": kind, "m": _log(rng, 1, min(8192, MOST_PRODUCTS // (n * k))), "n": n, "k": k,
                "fmt": rng.choice(("fp4", "fp8")), "bias": rng.random() < 0.4,
                "out": rng.choices(("bf16", "fp16", "fp32"), (6, 3, 1))[0]}
    hidden, ffn = rng.choice(BLOCKS)
    return {"kind": kind, "tokens": _log(rng, 1, min(2048, MOST_PRODUCTS // (3 * hidden * ffn))), "hidden": hidden,
            "ffn": ffn, "fmt": rng.choice(("fp4", "fp8"))}


# ----------------------------------------------------------------- plain forms
def _blocks(x):
    """[T, F] -> float32 [T, blocks, 32], the last block padded with zeros."""
    t, f = x.shape
    b = -(-f // 32)
    return torch.nn.functional.pad(x.float(), (0, 32 * b - f)).view(t, b, 32)


def _round_fp4(v):
    """|v| to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even code."""
    step = 0.5 * (1.0 + (v >= 2).float() + 2.0 * (v >= 4).float())
    return (torch.round(v / step) * step).clamp(max=6.0)


def _round_fp8(v):
    """|v| to the nearest e4m3 value, ties to the even code."""
    exponent = torch.frexp(v)[1].clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    return (torch.round(v / step) * step).clamp(max=448.0)


def _split(x, fmt):
    """Scale exponents [T, blocks] and the rounded values over the scale [T, blocks, 32] of a row's blocks."""
    v = _blocks(x)
    e = torch.frexp(v.abs().amax(2))[1] - 1 - (2 if fmt == "fp4" else 8)
    e = e.clamp(-127, 127)
    v = v / torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)[:, :, None]
    q = (_round_fp4 if fmt == "fp4" else _round_fp8)(v.abs())
    return e, torch.where(v < 0, -q, q)


def _values(x, fmt):
    """x [T, F] rounded to the format: float32 [T, F]."""
    e, q = _split(x, fmt)
    return (q * torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)[:, :, None]).flatten(1)[:, :x.shape[1]]


def _encode(x, fmt):
    """Codes and scale bytes of x, as a program keeps them."""
    e, q = _split(x, fmt)
    scales = (e + 127).to(torch.uint8)
    if fmt == "fp8":
        return q.flatten(1).to(torch.float8_e4m3fn), scales
    half = (q.abs() * 2).to(torch.uint8)          # 0 1 2 3 4 6 8 12 -> code 0 .. 7
    code = torch.where(half < 4, half, half // 2 + 2)
    code = torch.where(half == 12, 7, code) + 8 * (q < 0).to(torch.uint8)
    code = code.flatten(1).to(torch.uint8)
    return code[:, 0::2] + 16 * code[:, 1::2], scales


def _decode(codes, scales):
    """float32 [rows, 32 * blocks] of codes and scale bytes."""
    if codes.dtype == torch.uint8:
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), 2).long()].flatten(1)
    else:
        v = codes.float()
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return (v.view(v.shape[0], -1, 32) * s[:, :, None]).flatten(1)


def _norm(x, residual, weight):
    h = x.float() if residual is None else x.float() + residual.float()
    return h, h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * weight.float()


def _swiglu(x):
    gate, up = x.float().chunk(2, 1)
    return gate / (1.0 + torch.exp(-gate)) * up


# ----------------------------------------------------------------------- cases
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, tokens, features, dtype):
    """N(0, 1) with 0.5 % of the channels as outliers, x30."""
    x = torch.randn(tokens, features, generator=g, device="cuda")
    x[:, torch.randperm(features, generator=g, device="cuda")[: -(-features // 200)]] *= 30.0
    return x.to(dtype)


def _weight(g, n, k):
    return _encode(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5, "fp4")


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind == "quantize":
        s["x"] = _activations(g, case["tokens"], case["features"], DTYPES[case["dtype"]])
    elif kind == "norm":
        t, f, dtype = case["tokens"], case["features"], DTYPES[case["dtype"]]
        s["x"] = torch.randn(t, f, generator=g, device="cuda").to(dtype)
        s["residual"] = _activations(g, t, f, dtype) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(f, generator=g, device="cuda")).to(dtype)
    elif kind == "swiglu":
        s["x"] = (2.0 * torch.randn(case["tokens"], 2 * case["features"], generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    elif kind == "matmul":
        s["a"], s["sa"] = _encode(_activations(g, case["m"], case["k"], torch.float32), case["fmt"])
        s["b"], s["sb"] = _weight(g, case["n"], case["k"])
        s["bias"] = torch.randn(case["n"], generator=g, device="cuda").to(DTYPES[case["out"]]) if case["bias"] else None
    else:
        t, h, f = case["tokens"], case["hidden"], case["ffn"]
        s["x"] = torch.randn(t, h, generator=g, device="cuda").to(torch.bfloat16)
        s["residual"] = _activations(g, t, h, torch.bfloat16)
        s["weight"] = (1.0 + 0.1 * torch.randn(h, generator=g, device="cuda")).to(torch.bfloat16)
        s["up"], s["sup"] = _weight(g, 2 * f, h)
        s["down"], s["sdown"] = _weight(g, h, f)
    return s


def _run_own(s):
    import quant_ops_amd as qo

    case = s["case"]
    kind = case["kind"]
    fmt = "mx" + case["fmt"]
    if kind == "quantize":
        codes, scales = qo.mx_quantize(s["x"], fmt)
        return qo.mx_dequantize(codes, scales, features=case["features"], out_dtype=s["x"].dtype)
    if kind == "norm":
        got = qo.rms_norm_mx_quantize(s["x"], s["weight"], EPS, residual=s["residual"], fmt=fmt)
        return (qo.mx_dequantize(got[0], got[1], features=case["features"], out_dtype=torch.bfloat16),) + tuple(got[2:])
    if kind == "swiglu":
        codes, scales = qo.swiglu_mx_quantize(s["x"], fmt)
        return qo.mx_dequantize(codes, scales, features=case["features"], out_dtype=torch.bfloat16)
    if kind == "matmul":
        return qo.mx_matmul(s["a"], s["sa"], s["b"], s["sb"], bias=s["bias"], out_dtype=DTYPES[case["out"]])
    codes, scales, residual = qo.rms_norm_mx_quantize(s["x"], s["weight"], EPS, residual=s["residual"], fmt=fmt)
    gate_up = qo.mx_matmul(codes, scales, s["up"], s["sup"], out_dtype=torch.bfloat16)
    codes, scales = qo.swiglu_mx_quantize(gate_up, fmt)
    return qo.mx_matmul(codes, scales, s["down"], s["sdown"], out_dtype=torch.bfloat16), residual


def run(s):
    """One pass. Codes come back as the values they stand for; between the operators of the MLP block stand the
    bf16 tensors that a model holds there."""
    if own:
        return _run_own(s)
    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        return _values(s["x"], case["fmt"]).to(s["x"].dtype)
    if kind == "norm":
        h, y = _norm(s["x"], s["residual"], s["weight"])
        values = _values(y, case["fmt"]).to(torch.bfloat16)
        return (values,) if s["residual"] is None else (values, h.to(s["x"].dtype))
    if kind == "swiglu":
        return _values(_swiglu(s["x"]), case["fmt"]).to(torch.bfloat16)
    if kind == "matmul":
        out = _decode(s["a"], s["sa"]) @ _decode(s["b"], s["sb"]).t()
        return (out if s["bias"] is None else out + s["bias"].float()).to(DTYPES[case["out"]])
    h, y = _norm(s["x"], s["residual"], s["weight"])
    gate_up = (_values(y, case["fmt"]) @ _decode(s["up"], s["sup"]).t()).to(torch.bfloat16)
    out = _values(_swiglu(gate_up), case["fmt"]) @ _decode(s["down"], s["sdown"]).t()
    return out.to(torch.bfloat16), h.to(torch.bfloat16)


def work(case):
    size, kind = {"fp32": 4, "fp16": 2, "bf16": 2}, case["kind"]
    code = 0.5 + 1 / 32 if case["fmt"] == "fp4" else 1 + 1 / 32   # bytes of a coded value and its share of a scale
    if kind == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        out = size[case["out"]]
        return {"bytes": m * k * code + n * k * (0.5 + 1 / 32) + m * n * out + (n * out if case["bias"] else 0),
                "flops": 2 * m * n * k}
    t = case["tokens"]
    if kind == "mlp":
        h, f = case["hidden"], case["ffn"]
        return {"bytes": 4 * t * h * 2 + 2 * h + 3 * h * f * (0.5 + 1 / 32), "flops": 2 * t * 3 * h * f}
    f = case["features"]
    es = size[case["dtype"]]
    if kind == "quantize":
        return {"bytes": 2 * t * f * es, "flops": 4 * t * f}
    if kind == "norm":
        return {"bytes": t * f * (es * (3 if case["residual"] else 1) + 2) + f * es, "flops": 8 * t * f}
    return {"bytes": t * f * (2 * es + 2), "flops": 8 * t * f}


# -------------------------------------------------------- the definition in 64 bits
def _exact_values(x, fmt):
    t, f = x.shape
    b = -(-f // 32)
    v = torch.zeros(t, 32 * b, dtype=torch.float64, device=x.device)
    v[:, :f] = x
    v = v.reshape(t * b, 32)
    top, size = v.abs().max(1, keepdim=True).values, v.abs()
    scale = 2.0 ** (torch.floor(torch.log2(torch.where(top == 0, 1.0, top))) - (2 if fmt == "fp4" else 8))
    size = size / scale
    if fmt == "fp4":
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        half = (grid[1:] + grid[:-1]) / 2
        below = torch.bucketize(size, half)                   # a tie stays below
        at = torch.bucketize(size, half, right=True)          # a tie goes above
        q = grid[torch.where(below % 2 == 0, below, at)]      # to the even code
    else:
        e = torch.floor(torch.log2(torch.where(size == 0, 1.0, size))).clamp(min=-6)
        unit = 2.0 ** (e - 3)
        q = (torch.round(size / unit) * unit).clamp(max=448)
    return (torch.sign(v) * q * scale).reshape(t, 32 * b)[:, :f]


def _exact_decode(codes, scales):
    if codes.dtype == torch.uint8:
        nib = torch.stack((codes % 16, codes // 16), 2).flatten(1).double()
        sign, mag = 1 - 2 * torch.floor(nib / 8), nib % 8
        e, m = torch.floor(mag / 2), mag % 2
        v = sign * torch.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e - 1))
    else:
        v = codes.to(torch.float64)
    return v * (2.0 ** (scales.double() - 127)).repeat_interleave(32, 1)


def _exact_norm(s):
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
    return h, h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS) * s["weight"].double()


def _exact_swiglu(x):
    f = x.shape[1] // 2
    x = x.double()
    return x[:, :f] * torch.sigmoid(x[:, :f]) * x[:, f:]


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    fmt = case["fmt"]
    if kind == "quantize":
        return _exact_values(s["x"].double(), fmt)
    if kind == "norm":
        h, y = _exact_norm(s)
        return (_exact_values(y, fmt),) if s["residual"] is None else (_exact_values(y, fmt), h)
    if kind == "swiglu":
        return _exact_values(_exact_swiglu(s["x"]), fmt)
    if kind == "matmul":
        out = _exact_decode(s["a"], s["sa"]) @ _exact_decode(s["b"], s["sb"]).t().contiguous()
        return out if s["bias"] is None else out + s["bias"].double()
    h, y = _exact_norm(s)
    gate_up = (_exact_values(y, fmt) @ _exact_decode(s["up"], s["sup"]).t().contiguous()).to(torch.bfloat16)
    out = _exact_values(_exact_swiglu(gate_up), fmt) @ _exact_decode(s["down"], s["sdown"]).t().contiguous()
    return out, h
