"""The microscaled product's kernels, each at sizes that the host gives it (mx_plan,
dispatch_rules.h) with ragged edges: a case names its tile and the parts of its sum,
and test_mx_plan.py checks them on the CPU for 256 CUs. The bounds are those of
test_gpu_mx.py. The norm's and the dequantizer's variants follow."""
import pytest
import torch

import quant_ops_amd as qo
from oracle import mx_reference as om
from quant_ops_amd import capi
from test_gpu_mx import FMTS, _check_near, _check_product, _norm_error, _operand, _rows

pytestmark = pytest.mark.gpu

OUTS = (torch.bfloat16, torch.float32, torch.float16)

# M, N, blocks of 32 values; format; tile, parts
CASES = [
    (399, 16391, 33, "mxfp4", "256", 1),          # the last quad of k-steps holds one block
    (699, 16391, 17, "mxfp4", "256", 1),
    (1025, 11007, 1, "mxfp8", "256", 1),          # one block
    (399, 16391, 35, "mxfp8", "256", 1),
    (65, 16391, 1, "mxfp4", "128", 1),
    (129, 11007, 5, "mxfp4", "128", 1),
    (77, 16391, 35, "mxfp4", "128", 1),
    (65, 16391, 257, "mxfp4", "128", 1),          # 17 quads, one tile to a CU
    (77, 8201, 513, "mxfp4", "128", 2),           # 33: parts of 16 and 17
    (65, 8201, 448, "mxfp4", "128", 4),
    (65, 4097, 896, "mxfp4", "128", 8),
    (65, 8201, 3, "mxfp4", "128x64", 1),
    (77, 8201, 49, "mxfp4", "128x64", 1),
    (77, 2055, 300, "mxfp4", "128x64", 4),        # 19 quads, the last of 12 blocks
    (18, 41, 5, "mxfp4", "64", 1),
    (50, 130, 65, "mxfp4", "64", 1),
    (18, 4097, 257, "mxfp4", "64", 2),
    (33, 70, 193, "mxfp4", "64", 4),
    (18, 41, 300, "mxfp4", "64", 8),
    (65, 16391, 3, "mxfp8", "128", 1),
    (129, 11007, 1, "mxfp8", "128", 1),
    (77, 16391, 35, "mxfp8", "128", 1),
    (77, 8201, 257, "mxfp8", "128", 2),
    (65, 4097, 448, "mxfp8", "128", 4),
    (77, 2055, 513, "mxfp8", "128", 8),
    (65, 8201, 5, "mxfp8", "128x64", 1),
    (77, 8201, 49, "mxfp8", "128x64", 1),
    (18, 41, 5, "mxfp8", "64", 1),
    (50, 130, 65, "mxfp8", "64", 1),
    (18, 4097, 193, "mxfp8", "64", 2),            # 13 quads: parts of 6 and 7
    (33, 70, 129, "mxfp8", "64", 4),
    (18, 41, 300, "mxfp8", "64", 8),
]
# at most 16 rows: one quad to a wave and a's fragments kept, pairs of columns, 16 waves
STREAM = [(1, 41, 1), (16, 4097, 128), (9, 300, 97), (16, 8201, 130), (3, 8192, 449), (1, 77, 129), (16, 4097, 515)]


def _put(ts, gpu):
    return [t.to(gpu) for t in ts]


def _buffers(a, sa, gpu):
    """Codes and scales as the C interface takes them: scale rows at multiples of 16 bytes."""
    pad = torch.full((sa.shape[0], (sa.shape[1] + 15) // 16 * 16), 255, dtype=torch.uint8, device=gpu)   # NaN past the row
    pad[:, :sa.shape[1]] = sa.to(gpu)
    return a.to(gpu), pad[:, :sa.shape[1]]


@pytest.mark.parametrize("m,n,blocks,fmt,tile,parts", CASES)
def test_tile(gpu, m, n, blocks, fmt, tile, parts):
    (a, sa), (b, sb) = _operand(m, blocks, fmt, m + blocks, 116, 124), _operand(n, blocks, "mxfp4", n + blocks, 116, 124)
    da, dsa = _buffers(a, sa, gpu)
    db, dsb = _buffers(b, sb, gpu)
    g = torch.Generator().manual_seed(n)
    for i, out_dtype in enumerate(OUTS):
        print(f"[gpu-mx-tiles] {m} x {n} x {32 * blocks} {fmt} {out_dtype}: {tile} in {parts}", flush=True)
        bias = (8 * torch.randn(n, generator=g)).to(out_dtype) if i else None
        dbias = None if bias is None else bias.to(gpu)
        wide = torch.full((m, n + 8), 7.0, dtype=out_dtype, device=gpu)
        capi.mx_gemm(da, dsa, db, dsb, bias=dbias, out=wide[:, :n], workspace=True)
        torch.cuda.synchronize()
        assert bool((wide[:, n:] == 7.0).all())
        _check_product(wide[:, :n], a, sa, b, sb, bias)
        # contiguous rows, which leave odd rows unaligned where N is odd, and unpadded scales, which are copied
        got = qo.mx_matmul(da, dsa, db, sb.to(gpu), bias=dbias, out_dtype=out_dtype)
        assert torch.equal(got, wide[:, :n])
    if parts > 1:   # no workspace: one part
        _check_product(capi.mx_gemm(da, dsa, db, dsb, out_dtype=torch.float32), a, sa, b, sb)


@pytest.mark.parametrize("fmt,m,n,blocks", [("mxfp4", 399, 16391, 33), ("mxfp8", 399, 16391, 35), ("mxfp4", 65, 8201, 448),
                                            ("mxfp8", 77, 2055, 513), ("mxfp8", 65, 8201, 5)])
def test_nan_blocks_stay_in_their_rows(gpu, fmt, m, n, blocks):
    """A NaN block makes a row of a NaN and a column of b's, and nothing else changes."""
    (a, sa), (b, sb) = _operand(m, blocks, fmt, 1), _operand(n, blocks, "mxfp4", 2)
    a, sa, b, sb = _put((a, sa, b, sb), gpu)
    clean = qo.mx_matmul(a, sa, b, sb)
    rows, cols = [1, m // 2, m - 1], [0, n // 2, n - 1]
    sa[rows, [0, blocks // 2, blocks - 1]] = 255
    sb[cols, [blocks - 1, 0, blocks // 2]] = 255
    out = qo.mx_matmul(a, sa, b, sb)
    bad = torch.zeros(m, n, dtype=torch.bool, device=gpu)
    bad[rows], bad[:, cols] = True, True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,blocks", STREAM)
def test_few_rows(gpu, m, n, blocks, fmt):
    (a, sa), (b, sb) = _operand(m, blocks, fmt, m + blocks, 116, 124), _operand(n, blocks, "mxfp4", n + blocks, 116, 124)
    for i, out_dtype in enumerate(OUTS):
        print(f"[gpu-mx-tiles] {m} x {n} x {32 * blocks} {fmt} {out_dtype}", flush=True)
        bias = torch.linspace(-8, 8, n).to(out_dtype) if i else None
        out = qo.mx_matmul(*_put((a, sa, b, sb), gpu), bias=None if bias is None else bias.to(gpu), out_dtype=out_dtype)
        torch.cuda.synchronize()
        _check_product(out, a, sa, b, sb, bias)


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_far_apart(gpu, fmt):
    """Row strides above 4 MiB, which the tiles' 32-bit offsets do not take."""
    m, n, blocks, stride = 37, 45, 40, (1 << 22) + 16
    (a, sa), (b, sb) = _operand(m, blocks, fmt, 1), _operand(n, blocks, "mxfp4", 2)
    want = qo.mx_matmul(*_put((a, sa, b, sb), gpu), out_dtype=torch.float32)
    for far_a in (True, False):
        t = a if far_a else b
        raw = torch.empty((t.shape[0] - 1) * stride + t.shape[1], dtype=torch.uint8, device=gpu)
        far = raw.as_strided(tuple(t.shape), (stride, 1))
        far.copy_(t.view(torch.uint8))
        far = far.view(t.dtype)
        args = (far, sa.to(gpu), b.to(gpu), sb.to(gpu)) if far_a else (a.to(gpu), sa.to(gpu), far, sb.to(gpu))
        out = qo.mx_matmul(*args, out_dtype=torch.float32)
        torch.cuda.synchronize()
        _check_product(out, a, sa, b, sb)
        _check_product(want, a, sa, b, sb)


@pytest.mark.parametrize("fmt", FMTS)
def test_scale_rows_far_apart(gpu, fmt):
    """Rows of scales whose distances within a tile pass 32 bits."""
    m, n, blocks, stride = 130, 45, 40, 34 << 20
    (a, sa), (b, sb) = _operand(m, blocks, fmt, 1), _operand(n, blocks, "mxfp4", 2)
    raw = torch.empty((m - 1) * stride + 48, dtype=torch.uint8, device=gpu)
    far = raw.as_strided((m, blocks), (stride, 1))
    far.copy_(sa)
    out = qo.mx_matmul(a.to(gpu), far, b.to(gpu), sb.to(gpu), out_dtype=torch.float32)
    torch.cuda.synchronize()
    _check_product(out, a, sa, b, sb)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("feats", [4096, 4104, 8192, 8200, 16384, 16392, 24576, 24584, 32768, 32776, 4099, 8190, 33001])
def test_norm_lengths(gpu, feats, fmt):
    """Both sides of every line between the norm's variants; odd lengths."""
    x, res = _rows(5, feats, torch.bfloat16, feats), _rows(5, feats, torch.bfloat16, feats + 1)
    w = torch.linspace(-1.5, 1.5, feats)
    print(f"[gpu-mx-tiles] norm {feats} {fmt}", flush=True)
    codes, scales, h = qo.rms_norm_mx_quantize(x.to(gpu), w.to(gpu), residual=res.to(gpu), fmt=fmt)
    torch.cuda.synchronize()
    total, y = om.rms_norm(x.float() + res.float(), w, 1e-6)
    assert torch.equal(h.cpu(), total.to(torch.bfloat16))
    _check_near(y, _norm_error(feats), fmt, codes, scales)


@pytest.mark.parametrize("feats", [96, 4096])
def test_norm_unaligned(gpu, feats):
    """Inputs, weight and sum at odd element offsets equal the aligned call."""
    x, res = (_rows(6, feats, torch.float16, s).to(gpu) for s in (1, 2))
    w = torch.linspace(-1, 2, feats, device=gpu)
    want = qo.rms_norm_mx_quantize(x, w, residual=res)

    def shifted(t):
        out = torch.zeros(t.numel() + 1, dtype=t.dtype, device=gpu)[1:].view(t.shape)
        out.copy_(t)
        return out

    for part in range(4):
        args = [shifted(t) if part in (i, 3) else t for i, t in enumerate((x, w, res))]
        got = qo.rms_norm_mx_quantize(args[0], args[1], residual=args[2])
        # another variant adds the squares in another order: the sum is exact, codes within the bound
        assert torch.equal(got[2], want[2])
        _check_near(om.rms_norm(x.cpu().float() + res.cpu().float(), w.cpu(), 1e-6)[1], _norm_error(feats), "mxfp8", got[0],
                    got[1])
    out = torch.zeros(x.numel() + 1, dtype=x.dtype, device=gpu)[1:].view(x.shape)
    got = capi.rms_norm_mx_quantize(x, w, residual=res, residual_out=out)
    assert torch.equal(got[2], want[2]) and out.data_ptr() == got[2].data_ptr()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("out_dtype", OUTS)
@pytest.mark.parametrize("tokens,feats", [(1, 1), (1, 33), (3, 100), (5, 4097), (700, 4096), (300, 40000)])
def test_dequantize(gpu, tokens, feats, out_dtype, fmt):
    """Exact up to the output's one rounding, from scales in rows of a wider buffer; calls
    below and above the size from which stores pass the cache."""
    blocks = -(-feats // 32)
    codes, scales = _operand(tokens, blocks, fmt, feats, 100, 150)
    wide = torch.full((tokens, blocks + 5), 255, dtype=torch.uint8, device=gpu)
    wide[:, 3:3 + blocks] = scales.to(gpu)
    print(f"[gpu-mx-tiles] dequantize {tokens} x {feats} {fmt} {out_dtype}", flush=True)
    out = qo.mx_dequantize(codes.to(gpu), wide[:, 3:3 + blocks], feats, out_dtype)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), om.values(codes, scales)[:, :feats].to(out_dtype))
