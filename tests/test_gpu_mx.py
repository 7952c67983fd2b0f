"""GPU tests of the microscaled operators against their definition in 64 bits.

Quantizing and dequantizing take no arithmetic that rounds, so they are exact.
Where a float32 y is quantized (norm, gate), y's relative error is at most d
(below), so a scale byte must be that of the largest magnitude times some
factor in [1 - d, 1 + d], and a code the rounding of its value times such a
factor: both are monotone, so the two ends bracket them."""
import pytest
import torch

import quant_ops_amd as qo
from oracle import mx_reference as om
from quant_ops_amd import capi

pytestmark = pytest.mark.gpu

FMTS = ("mxfp4", "mxfp8")
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
U = 2.0 ** -24   # float32's unit roundoff


def _say(msg):
    print(f"[gpu-mx] {msg}", flush=True)


def _rows(tokens, feats, dtype, seed):
    """N(0, 1) rows of very different sizes with outliers; some blocks zero."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, feats, generator=g)
    x *= torch.exp2(torch.randint(-6, 7, (tokens, 1), generator=g).float())
    x[torch.rand(tokens, feats, generator=g) < 0.01] *= 30.0
    if feats > 40:
        x[::3, 32:64] = 0.0
    return x.to(dtype)


def _signed(v):
    """Values with the sign of zeros visible."""
    return torch.stack((v, torch.signbit(v).double()))


def _check_exact(x, fmt, codes, scales):
    q, byte = om.quantize(x.cpu().double(), fmt)
    assert codes.shape == (x.shape[0], q.shape[1] * (16 if fmt == "mxfp4" else 32)) and scales.shape == byte.shape
    assert torch.equal(scales.cpu().long(), byte)
    assert torch.equal(_signed(om.code_values(codes)), _signed(q))


def _check_near(y, d, fmt, codes, scales):
    """codes and scales of a float32 computation of y (float64) with relative error d."""
    v, got = om.blocks_of(y), scales.cpu().long()
    top = v.abs().amax(2)
    lo, hi = om.scale_bytes(top * (1 - d), fmt), om.scale_bytes(top * (1 + d), fmt)
    assert bool(((got == lo) | (got == hi)).all())
    s = torch.ldexp(torch.ones_like(top), got - 127)[:, :, None]
    c = om.code_values(codes)
    a, b = om.round_codes(v * (1 - d) / s, fmt), om.round_codes(v * (1 + d) / s, fmt)
    assert bool(((torch.minimum(a, b) <= c) & (c <= torch.maximum(a, b))).all())


SIZES = [(1, 1), (1, 31), (1, 32), (2, 33), (3, 64), (5, 100), (1, 4096), (7, 4096), (16, 1000), (33, 4104), (3, 14336),
         (300, 264), (1021, 72), (2, 32800)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,feats", SIZES)
def test_quantize_exact(gpu, tokens, feats, dtype, fmt):
    x = _rows(tokens, feats, dtype, seed=tokens + feats).to(gpu)
    codes, scales = qo.mx_quantize(x, fmt)
    torch.cuda.synchronize()
    _check_exact(x, fmt, codes, scales)
    for out_dtype in DTYPES:
        y = qo.mx_dequantize(codes, scales, features=feats, out_dtype=out_dtype)
        assert y.dtype == out_dtype and y.shape == x.shape
        assert torch.equal(y.cpu(), om.values(codes, scales)[:, :feats].to(out_dtype))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_every_exponent_and_tie(gpu, fmt):
    """Blocks at every float32 exponent, subnormal ones too; every code, every tie and their neighbours."""
    if fmt == "mxfp4":
        grid = om.GRID4
    else:
        grid = torch.arange(0, 127).to(torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    points = torch.cat([grid, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), grid[-1:] * 1.1])
    top = 4.0 if fmt == "mxfp4" else 256.0   # holds the block's exponent
    rows = []
    for i in range(0, len(points), 31):
        p = points[i:i + 31]
        rows.append(torch.cat([torch.tensor([top]), p, torch.zeros(31 - len(p))]))
    base = torch.stack(rows).double()
    base = torch.cat([base, -base])
    exps = range(-146, 119) if fmt == "mxfp8" else range(-149, 125)
    x = torch.cat([torch.ldexp(base, torch.tensor(e)) for e in exps]).float()
    codes, scales = qo.mx_quantize(x.to(gpu), fmt)
    torch.cuda.synchronize()
    _check_exact(x, fmt, codes, scales)
    y = qo.mx_dequantize(codes, scales)
    assert torch.equal(y.cpu(), om.values(codes, scales).float())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_non_finite_blocks(gpu, dtype, fmt):
    x = _rows(8, 160, dtype, seed=5)
    x[0, 3], x[1, 40], x[2, 159], x[3, 64:96] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[4, 32:64] = torch.finfo(dtype).max
    x[5, 32:64] = torch.finfo(dtype).tiny
    x[6] = -0.0
    codes, scales = qo.mx_quantize(x.to(gpu), fmt)
    torch.cuda.synchronize()
    _check_exact(x, fmt, codes, scales)
    y = qo.mx_dequantize(codes, scales).cpu()
    bad = torch.zeros(8, 5, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 4] = bad[3, 2] = True
    assert torch.equal(torch.isnan(y).view(8, 5, 32), bad[:, :, None].expand(8, 5, 32))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_strides_and_leading_dimensions(gpu, fmt):
    wide = _rows(12, 600, torch.bfloat16, seed=9).to(gpu)
    for x in (wide[:, 1:501], wide[::2, 3:259], wide.t()[5:105], wide[:1].expand(6, 600), wide[3, 7:7 + 64][None]):
        codes, scales = qo.mx_quantize(x, fmt)
        torch.cuda.synchronize()
        _check_exact(x, fmt, codes, scales)
    x = wide.view(3, 4, 600)
    codes, scales = qo.mx_quantize(x, fmt)
    assert codes.shape[:2] == (3, 4) and scales.shape == (3, 4, 19)
    assert torch.equal(qo.mx_dequantize(codes, scales, features=600).view(12, 600),
                       qo.mx_dequantize(*qo.mx_quantize(wide, fmt), features=600))


# y's relative error: the sum of F squares, in float32 by threads of at most F / 256
# + 8 terms and then pairwise (10 levels, 16 wave sums), its root (half of that), the
# mean, the root, the reciprocal and the three products, one rounding each.
def _norm_error(feats):
    return ((feats / 256 + 8 + 10 + 16) / 2 + 8) * U


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_residual", (False, True))
@pytest.mark.parametrize("tokens,feats", SIZES + [(3, 8192), (2, 28672), (600, 512), (1, 70000)])
def test_norm(gpu, tokens, feats, with_residual, dtype, fmt):
    x = _rows(tokens, feats, dtype, seed=3 * tokens + feats)
    res = _rows(tokens, feats, dtype, seed=7 * tokens + feats) if with_residual else None
    g = torch.Generator().manual_seed(feats)
    w = (1 + 0.2 * torch.randn(feats, generator=g)).to(DTYPES[(tokens + feats) % 3])
    got = qo.rms_norm_mx_quantize(x.to(gpu), w.to(gpu), 1e-5, residual=None if res is None else res.to(gpu), fmt=fmt)
    torch.cuda.synchronize()
    # the addition of float32 inputs rounds: the norm is of the rounded sum, as it stands
    h32 = x.float() if res is None else x.float() + res.float()
    _check_near(om.rms_norm(h32, w, 1e-5)[1], _norm_error(feats), fmt, got[0], got[1])
    assert len(got) == (3 if with_residual else 2)
    if with_residual:
        assert torch.equal(got[2].cpu(), h32.to(dtype))


def test_norm_zero_and_non_finite_rows(gpu):
    x = _rows(6, 4096, torch.bfloat16, seed=1)
    x[1], x[2, 5], x[3, 7] = 0.0, float("nan"), float("inf")
    w = torch.ones(4096, dtype=torch.bfloat16)
    codes, scales = qo.rms_norm_mx_quantize(x.to(gpu), w.to(gpu), 1e-6)
    y = qo.mx_dequantize(codes, scales).cpu()
    assert bool((y[1] == 0).all()) and bool((scales[1] == 0).all())
    assert bool(torch.isnan(y[2]).all())
    # an infinite value: its own quotient is NaN (inf / inf), the others are 0
    assert bool(torch.isnan(y[3, :32]).all()) and bool((y[3, 32:] == 0).all())
    for r in (0, 4, 5):
        assert bool(torch.isfinite(y[r]).all())


def test_norm_strides_and_residual_in_place(gpu):
    wide, res = _rows(9, 1200, torch.float16, seed=2).to(gpu), _rows(9, 1200, torch.float16, seed=3).to(gpu)
    w = torch.randn(1111, device=gpu)
    x, r = wide[:, 5:1116], res[:, 77:1188]
    got = qo.rms_norm_mx_quantize(x, w, residual=r)
    want = qo.rms_norm_mx_quantize(x.contiguous(), w, residual=r.contiguous())
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # the C ABI may write the sum over the residual
    stream = capi.rms_norm_mx_quantize(x.contiguous(), w, residual=(same := r.contiguous()), residual_out=same)
    torch.cuda.synchronize()
    assert torch.equal(same, want[2])
    assert torch.equal(stream[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(stream[1], want[1])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,feats", SIZES)
def test_swiglu(gpu, tokens, feats, dtype, fmt):
    g = torch.Generator().manual_seed(tokens + feats)
    x = (3 * torch.randn(tokens, 2 * feats, generator=g)).to(dtype)
    codes, scales = qo.swiglu_mx_quantize(x.to(gpu), fmt)
    torch.cuda.synchronize()
    # exp (2 units), its argument exact, the sum, the quotient and the product
    _check_near(om.swiglu(x.float()), 8 * U, fmt, codes, scales)


def test_swiglu_large_gates(gpu):
    """One gate to a block; float32's exp is infinite from 89 on, so such gates give zeros."""
    g = torch.tensor([-1000.0, -200.0, -90.0, -87.0, -20.0, 0.0, 20.0, 90.0, 1000.0, -0.0, float("inf"), float("nan")])
    x = torch.cat([g[:, None].expand(-1, 32), torch.full((len(g), 32), 1.5)], 1).contiguous()
    codes, scales = (t.cpu() for t in qo.swiglu_mx_quantize(x.to(gpu), "mxfp8"))
    y = (g / (1 + torch.exp(-g)) * 1.5)[:, None].double().expand(-1, 32)
    # exp(87): 1 unit for its argument's rounding at base 2, times 87 * log2(e)
    _check_near(y[:-2], 140 * U, "mxfp8", codes[:-2], scales[:-2])
    assert bool((scales[-2:] == 255).all()) and bool((codes[-2:].view(torch.uint8) == 0).all())


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_swiglu_largest_gates(gpu, dtype):
    """Gates up to the type's largest, where g log2(e) leaves float32: silu(g) is g, or 0 below."""
    top = torch.finfo(dtype).max
    g = torch.tensor([128.0, 1e10, 2.0 ** 127, 2.3e38, 2.4e38, 3e38, top, -1e10, -2.0 ** 127, -3e38, -top]).to(dtype)
    x = torch.cat([g[:, None].expand(-1, 32), torch.full((len(g), 32), 2.0 ** -10, dtype=dtype)], 1).contiguous()
    codes, scales = qo.swiglu_mx_quantize(x.to(gpu), "mxfp8")
    torch.cuda.synchronize()
    y = (g.double().clamp(min=0) * 2.0 ** -10)[:, None].expand(-1, 32)
    _check_near(y, 8 * U, "mxfp8", codes, scales)


def _operand(rows, blocks, fmt, seed, lo=118, hi=136):
    """Random codes (every finite one) and scale bytes."""
    g = torch.Generator().manual_seed(seed)
    scales = torch.randint(lo, hi, (rows, blocks), generator=g).to(torch.uint8)
    if fmt == "mxfp4":
        return torch.randint(0, 256, (rows, 16 * blocks), generator=g).to(torch.uint8), scales
    c = torch.randint(0, 254, (rows, 32 * blocks), generator=g)
    return torch.where(c >= 127, c + 1, c).to(torch.uint8).view(torch.float8_e4m3fn), scales


def _exponents8(codes, scales, least):
    """2^(largest exponent) of each eight consecutive values, times their scale; subnormal
    codes have the least normal exponent, groups of zeros none."""
    v = om.code_values(codes).abs()
    e = torch.where(v > 0, torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp(min=least)), 0.0)
    e = e.view(v.shape[0], v.shape[1], 4, 8).amax(3)
    byte = scales.cpu().long()
    return (e * torch.ldexp(torch.ones_like(byte, dtype=torch.float64), byte - 127)[:, :, None]).flatten(1)


def _check_product(out, a, sa, b, sb, bias=None):
    """|out - exact| against: one rounding to the output type; the float32 sums over k-steps (their
    halves, the split's parts), at most a unit of the terms' magnitudes each and four units within
    a step; and for 16-bit outputs of FP8 codes what the matrix core drops of each eight products,
    seven terms' bits below 2^-13 of 2^(largest exponent of the eight a) 2^(that of the b)."""
    want, mag = om.matmul(a, sa, b, sb)
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    steps = 2 * -(-sa.shape[1] // 4) + 16
    drop = 0.0
    if a.dtype != torch.uint8 and out.dtype != torch.float32:
        drop = 7 * 2.0 ** -13 * (_exponents8(a, sa, -6) @ _exponents8(b, sb, 0).t())
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[out.dtype]
    least = 2.0 ** -24 if out.dtype == torch.float16 else 0.0
    bound = unit * want.abs() + (1 + unit) * ((2.0 ** -22 + 2 * U * steps) * mag + drop) + least
    got = out.cpu().double()
    # infinite: only where a value within the bound rounds past the type's largest (by half its last unit)
    top = torch.finfo(out.dtype).max * (1 + unit / 2)
    fine = torch.where(torch.isinf(got), (torch.sign(got) == torch.sign(want)) & (want.abs() + bound >= top),
                       (got - want).abs() <= bound)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert bool((fine | nan).all()), f"{int((~fine & ~nan).sum())} of {fine.numel()} outputs off"


PRODUCTS = [(1, 1, 32), (1, 16, 128), (1, 4096, 512), (2, 5, 64), (15, 17, 96), (16, 33, 160), (17, 64, 4096), (33, 130, 544),
            (64, 100, 2080), (65, 257, 1056), (127, 129, 256), (128, 256, 512), (130, 255, 640), (200, 512, 128),
            (256, 256, 1024), (257, 300, 4128), (300, 513, 96), (512, 514, 2048), (1000, 24, 4096), (5, 1000, 14336)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul(gpu, m, n, k, fmt):
    (a, sa), (b, sb) = _operand(m, k // 32, fmt, m + k), _operand(n, k // 32, "mxfp4", n + k + 1)
    g = torch.Generator().manual_seed(n)
    _say(f"{m} x {n} x {k} {fmt}")
    for i, out_dtype in enumerate((torch.bfloat16, torch.float32, torch.float16)):
        bias = (8 * torch.randn(n, generator=g)).to(out_dtype) if (m + i) % 2 else None
        out = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), bias=None if bias is None else bias.to(gpu),
                           out_dtype=out_dtype)
        torch.cuda.synchronize()
        assert out.shape == (m, n) and out.dtype == out_dtype
        _check_product(out, a, sa, b, sb, bias)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(1, 70, 96), (17, 40, 544), (100, 300, 1056), (300, 520, 640)])
def test_matmul_fp16_range(gpu, m, n, k, fmt):
    """Outputs inside float16's range."""
    (a, sa), (b, sb) = _operand(m, k // 32, fmt, m + k, 116, 122), _operand(n, k // 32, "mxfp4", n + k, 116, 122)
    out = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), out_dtype=torch.float16)
    assert bool(torch.isfinite(out).all())
    _check_product(out, a, sa, b, sb)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (100, 300, 1056), (300, 520, 640)])
def test_matmul_nan_scales_stay_in_their_rows(gpu, m, n, k, fmt):
    """A NaN block of a row of a makes that row NaN, one of b its column; the others do not change."""
    (a, sa), (b, sb) = _operand(m, k // 32, fmt, 1), _operand(n, k // 32, "mxfp4", 2)
    clean = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), out_dtype=torch.float32).cpu()
    rows, cols = [0, m // 2, m - 1], [1, n - 1]
    sa[rows, [0, k // 32 - 1, k // 64]] = 255
    sb[cols, [k // 64, k // 32 - 1]] = 255
    out = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), out_dtype=torch.float32).cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[rows], bad[:, cols] = True, True
    assert torch.equal(torch.isnan(out), bad)
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("fmt", FMTS)
def test_matmul_extreme_scales(gpu, fmt):
    """Scale bytes 0 and 254 and products that leave float32's range at either end."""
    (a, sa), (b, sb) = _operand(20, 8, fmt, 3), _operand(40, 8, "mxfp4", 4)
    a = a.clone()
    a.view(torch.uint8)[:, 0] = 0x22 if fmt == "mxfp4" else 0x38   # 1.0
    sa[:], sb[:] = 0, 254
    sa[1], sb[1] = 254, 0
    out = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu), out_dtype=torch.float32).cpu()
    want, mag = om.matmul(a, sa, b, sb)
    small = mag < 2.0 ** 100
    tol = 2.0 ** -20 * mag + 2.0 ** -126
    assert bool(((out.double() - want).abs() <= tol)[small].all())
    assert bool((~torch.isfinite(out))[mag > 2.0 ** 140].all())


@pytest.mark.parametrize("fmt", FMTS)
def test_matmul_strides_and_offsets(gpu, fmt):
    """Rows of wider buffers, unaligned starts (copied), strided scales, a strided bias."""
    width = 1 if fmt == "mxfp8" else 2
    (a, sa), (b, sb) = _operand(50, 40, fmt, 5), _operand(140, 40, "mxfp4", 6)
    a, sa, b, sb = (t.to(gpu) for t in (a, sa, b, sb))
    # blocks 4 .. 23 of rows 1, 3, ..
    va, vsa = a[1::2, 4 * 32 // width:24 * 32 // width], sa[1::2, 4:24]
    vb, vsb = b[1:, 64:384], sb[1:, 4:24]
    bias = torch.randn(139, 3, device=gpu)[:, 1]
    out = qo.mx_matmul(va, vsa, vb, vsb, bias=bias, out_dtype=torch.float32)
    same = qo.mx_matmul(va.contiguous(), vsa.contiguous(), vb.contiguous(), vsb.contiguous(), bias=bias.contiguous(),
                        out_dtype=torch.float32)
    assert torch.equal(out, same)
    _check_product(out, va.contiguous(), vsa, vb.contiguous(), vsb, bias.cpu())
    raw = torch.zeros(b.numel() + 1, dtype=torch.uint8, device=gpu)
    off = raw[1:].view(140, 640)
    off.copy_(b)
    assert torch.equal(qo.mx_matmul(a, sa, off, sb), qo.mx_matmul(a, sa, b, sb))
    assert torch.equal(qo.mx_matmul(a.view(5, 10, -1), sa.view(5, 10, -1), b, sb).view(50, 140), qo.mx_matmul(a, sa, b, sb))


def test_empty_calls(gpu):
    x = torch.zeros(0, 64, device=gpu)
    for fmt in FMTS:
        codes, scales = qo.mx_quantize(x, fmt)
        assert codes.shape[0] == 0 and scales.shape == (0, 2)
        codes, scales = qo.mx_quantize(torch.zeros(4, 0, device=gpu), fmt)
        assert codes.shape == (4, 0) and scales.shape == (4, 0)
        assert qo.mx_dequantize(codes, scales).shape == (4, 0)
        codes, scales = qo.swiglu_mx_quantize(torch.zeros(0, 64, device=gpu), fmt)
        assert scales.shape == (0, 1)
        assert qo.rms_norm_mx_quantize(x, torch.ones(64, device=gpu), residual=x, fmt=fmt)[2].shape == (0, 64)
    b, sb = (t.to(gpu) for t in _operand(7, 2, "mxfp4", 1))
    assert qo.mx_matmul(b[:0], sb[:0], b, sb).shape == (0, 7)
    assert qo.mx_matmul(b, sb, b[:0], sb[:0]).shape == (7, 0)
    # no blocks: the sum is empty
    none = torch.zeros(3, 0, dtype=torch.uint8, device=gpu)
    bias = torch.tensor([1.0, -2.0, 3.0], device=gpu)
    assert torch.equal(qo.mx_matmul(none, none, none, none, bias=bias, out_dtype=torch.float32), bias.expand(3, 3))


def test_past_32_bits(gpu):
    """Rows whose elements, and outputs whose positions, lie past 2^31."""
    tokens, feats = 70000, 32768
    x = torch.zeros(tokens, feats, dtype=torch.bfloat16, device=gpu)
    tail = _rows(5, feats, torch.bfloat16, seed=8)
    x[-5:] = tail.to(gpu)
    for fmt in FMTS:
        codes, scales = qo.mx_quantize(x, fmt)
        torch.cuda.synchronize()
        _check_exact(tail, fmt, codes[-5:], scales[-5:])
        y = qo.mx_dequantize(codes, scales, out_dtype=torch.bfloat16)
        assert torch.equal(y[-5:].cpu(), om.values(codes[-5:], scales[-5:]).to(torch.bfloat16))
        del y
    got = qo.rms_norm_mx_quantize(x, torch.ones(feats, device=gpu), residual=x)
    _check_near(om.rms_norm(2 * tail.float(), torch.ones(feats), 1e-6)[1], _norm_error(feats), "mxfp8", got[0][-5:], got[1][-5:])
    del got, x
    (a, sa), (b, sb) = _operand(tokens, 1, "mxfp8", 1), _operand(feats, 1, "mxfp4", 2)
    out = qo.mx_matmul(a.to(gpu), sa.to(gpu), b.to(gpu), sb.to(gpu))
    _check_product(out[-3:], a[-3:], sa[-3:], b, sb)


def test_side_stream_and_graph(gpu):
    """On a stream that is not the tensors' own, and captured: replays equal eager calls."""
    x = _rows(24, 4096, torch.bfloat16, seed=4).to(gpu)
    res = _rows(24, 4096, torch.bfloat16, seed=5).to(gpu)
    w = torch.ones(4096, dtype=torch.bfloat16, device=gpu)
    b, sb = (t.to(gpu) for t in _operand(2 * 512, 128, "mxfp4", 6, 110, 121))
    d, sd = (t.to(gpu) for t in _operand(300, 16, "mxfp4", 7, 110, 121))

    def step():
        codes, scales, h = qo.rms_norm_mx_quantize(x, w, residual=res)
        codes, scales = qo.swiglu_mx_quantize(qo.mx_matmul(codes, scales, b, sb))
        return qo.mx_matmul(codes, scales, d, sd), h

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = step()
    torch.cuda.synchronize()
    keep = x.clone()
    for rep in range(4):
        x.copy_(keep * (1 + rep % 2))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, eager)), f"replay {rep}"
    x.copy_(keep)


def test_host_tensors_equal_the_gpu(gpu):
    """The PyTorch forms of host tensors give the kernels' codes where no arithmetic rounds."""
    for fmt in FMTS:
        x = _rows(9, 1000, torch.float16, seed=6)
        host, dev = qo.mx_quantize(x, fmt), qo.mx_quantize(x.to(gpu), fmt)
        assert all(torch.equal(h.view(torch.uint8), d.cpu().view(torch.uint8)) for h, d in zip(host, dev))
        assert torch.equal(qo.mx_dequantize(*host, features=1000), qo.mx_dequantize(*dev, features=1000).cpu())


def test_gpu_refusals(gpu):
    x = torch.zeros(4, 64, device=gpu)
    b = torch.zeros(8, 32, dtype=torch.uint8, device=gpu)
    sb = torch.zeros(8, 2, dtype=torch.uint8, device=gpu)
    w = torch.ones(64, device=gpu)
    bad = [
        lambda: qo.mx_quantize(x.double()),
        lambda: qo.mx_quantize(x.int()),
        lambda: qo.mx_quantize(x, "mxfp6"),
        lambda: qo.mx_dequantize(b, sb[:, :1]),
        lambda: qo.mx_dequantize(b, sb, features=65),
        lambda: qo.mx_dequantize(b, sb, features=32),
        lambda: qo.mx_dequantize(b.int(), sb),
        lambda: qo.mx_dequantize(b, sb.int()),
        lambda: qo.mx_dequantize(b, sb, out_dtype=torch.float64),
        lambda: qo.mx_dequantize(b, sb.cpu()),
        lambda: qo.rms_norm_mx_quantize(x, w[:63]),
        lambda: qo.rms_norm_mx_quantize(x, w.double()),
        lambda: qo.rms_norm_mx_quantize(x, w.cpu()),
        lambda: qo.rms_norm_mx_quantize(x, w, residual=x[:3]),
        lambda: qo.rms_norm_mx_quantize(x, w, residual=x.half()),
        lambda: qo.rms_norm_mx_quantize(x, w, residual=x.cpu()),
        lambda: qo.swiglu_mx_quantize(x[:, :63]),
        lambda: qo.swiglu_mx_quantize(x.double()),
        lambda: qo.mx_matmul(b, sb, b[:, :16], sb[:, :1]),
        lambda: qo.mx_matmul(b, sb[:4], b, sb),
        lambda: qo.mx_matmul(b.float(), sb, b, sb),
        lambda: qo.mx_matmul(b, sb, torch.zeros(8, 64, device=gpu).to(torch.float8_e4m3fn), sb),
        lambda: qo.mx_matmul(b, sb, b, sb, bias=torch.zeros(7, device=gpu)),
        lambda: qo.mx_matmul(b, sb, b, sb, bias=torch.zeros(8)),
        lambda: qo.mx_matmul(b, sb, b, sb, out_dtype=torch.float64),
        lambda: qo.mx_matmul(b, sb, b.cpu(), sb),
        lambda: qo.mx_matmul(b, sb.float(), b, sb),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was accepted")
