"""Host side of the microscaled operators (no GPU): the PyTorch forms against the
definition in 64 bits, the C ABI's checks, the fakes, and the oracle's own grids."""
import ctypes

import pytest
import torch

import quant_ops_amd as qo
from oracle import mx_reference as om
from quant_ops_amd import capi

FMTS = ("mxfp4", "mxfp8")


def test_oracle_grids():
    # the FP8 grid is torch's e4m3; the FP4 grid its definition: s e e m, bias 1, subnormals 0 and 1/2
    every = torch.arange(0, 127).to(torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(om.round_codes(every, "mxfp8"), every)
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.randn(4000, generator=g).double() * 100, (every[1:] + every[:-1]) / 2])
    assert torch.equal(om.round_codes(v, "mxfp8"), v.clamp(-448, 448).float().to(torch.float8_e4m3fn).double())
    want = [m / 2 if e == 0 else (1 + m / 2) * 2.0 ** (e - 1) for e in range(4) for m in range(2)]
    assert om.GRID4.tolist() == want
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -5.0])
    assert om.round_codes(ties.double(), "mxfp4").tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -4]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("tokens,feats", [(1, 1), (3, 32), (2, 33), (5, 100), (0, 64), (4, 0), (7, 1000)])
def test_quantize_host(tokens, feats, dtype, fmt):
    g = torch.Generator().manual_seed(feats)
    x = (torch.randn(tokens, feats, generator=g) * torch.exp2(torch.randint(-8, 9, (tokens, 1), generator=g).float())).to(dtype)
    if feats > 64:
        x[0, 5], x[1, 40], x[2, :32] = float("nan"), float("inf"), 0.0
    codes, scales = qo.mx_quantize(x, fmt)
    q, byte = om.quantize(x.double(), fmt)
    assert torch.equal(scales.long(), byte) and torch.equal(om.code_values(codes), q)
    y = qo.mx_dequantize(codes, scales, features=feats, out_dtype=dtype)
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(om.values(codes, scales)[:, :feats].to(dtype)))


def test_quantize_host_extremes():
    x = torch.tensor([[2.0 ** -149] * 32, [2.0 ** -126] * 32, [3.4e38] * 32, [0.0] * 32])
    for fmt in FMTS:
        codes, scales = qo.mx_quantize(x, fmt)
        q, byte = om.quantize(x.double(), fmt)
        assert torch.equal(scales.long(), byte) and torch.equal(om.code_values(codes), q)


@pytest.mark.parametrize("fmt", FMTS)
def test_path_host(fmt):
    """Norm, product, gate and product on host tensors against 64 bits on the same codes."""
    g = torch.Generator().manual_seed(3)
    x, res = torch.randn(2, 5, 96, generator=g), torch.randn(2, 5, 96, generator=g)
    w = 1 + 0.1 * torch.randn(96, generator=g)
    up, down = (qo.mx_quantize(torch.randn(n, k, generator=g) / 8, "mxfp4") for n, k in ((80, 96), (33, 40)))
    codes, scales, h = qo.rms_norm_mx_quantize(x, w, 1e-5, residual=res, fmt=fmt)
    assert torch.equal(h, x + res) and codes.shape[:2] == (2, 5)
    y = om.rms_norm((x + res).view(10, 96), w, 1e-5)[1]
    err = (qo.mx_dequantize(codes, scales).view(10, 96).double() - y).abs()
    assert bool((err <= om.blocks_of(y).abs().amax(2).repeat_interleave(32, 1) / (4 if fmt == "mxfp4" else 8)).all())
    gate_up = qo.mx_matmul(codes, scales, *up, out_dtype=torch.float32)
    want = om.matmul(codes.view(10, -1), scales.view(10, -1), *up)[0]
    assert torch.allclose(gate_up.view(10, 80).double(), want, rtol=1e-5, atol=1e-5)
    codes, scales = qo.swiglu_mx_quantize(gate_up, fmt)
    bias = torch.randn(33, generator=g)
    out = qo.mx_matmul(codes, scales, *down, bias=bias)
    assert out.shape == (2, 5, 33) and out.dtype == torch.bfloat16
    want = om.matmul(codes.view(10, -1), scales.view(10, -1), *down)[0] + bias.bfloat16().double()
    assert torch.allclose(out.view(10, 33).double(), want, rtol=2.0 ** -8, atol=1e-4)


def test_host_refusals():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="mxfp"):
        qo.mx_quantize(x, "fp4")
    with pytest.raises(ValueError, match="residual"):
        qo.rms_norm_mx_quantize(x, torch.ones(64), residual=x[:1])
    with pytest.raises(ValueError, match="halves"):
        qo.swiglu_mx_quantize(x[:, :63])
    with pytest.raises(AssertionError, match="blocks"):
        qo.mx_dequantize(*qo.mx_quantize(x), features=30)


def _p(v):
    return ctypes.c_void_p(v)


def test_c_abi_checks():
    """Every refusal of the C entry points comes before a launch (the addresses are never read)."""
    lib = capi.lib()
    A = 4096   # an aligned, unused address
    quantize = lambda x=A, dt=1, t=4, f=64, ld=64, fmt=0, c=A, s=A, sl=2: lib.qo_mx_quantize(_p(x), dt, t, f, ld, fmt, _p(c), _p(s), sl, _p(None))  # noqa: E731
    assert quantize(t=0) == 0 and quantize(f=0) == 0
    assert quantize(t=-1) == 2 and quantize(f=2 ** 31, sl=2 ** 26) == 2 and quantize(ld=63) == 2 and quantize(sl=1) == 2
    assert quantize(dt=3) == 3 and quantize(fmt=2) == 3 and quantize(fmt=-1) == 3
    assert quantize(x=None) == 1 and quantize(c=None) == 1 and quantize(s=None) == 1
    assert quantize(c=A + 4) == 4 and b"aligned" in lib.qo_last_error()
    deq = lambda c=A, s=A, fmt=0, t=4, f=64, o=A, dt=0: lib.qo_mx_dequantize(_p(c), _p(s), 2, fmt, t, f, _p(o), dt, _p(None))  # noqa: E731
    assert deq(t=0) == 0 and deq(f=-1) == 2 and deq(dt=4) == 3 and deq(fmt=7) == 3 and deq(o=None) == 1 and deq(c=A + 2) == 4
    norm = lambda x=A, r=None, dt=1, t=4, f=64, ld=64, rld=64, w=A, wd=0, fmt=1, c=A, s=A, ro=None: lib.qo_rms_norm_mx_quantize(  # noqa: E731
        _p(x), _p(r), dt, t, f, ld, rld, _p(w), wd, 1e-6, fmt, _p(c), _p(s), 2, _p(ro), _p(None))
    assert norm(t=0) == 0 and norm(ld=63) == 2 and norm(r=A, rld=63, ro=A) == 2 and norm(wd=3) == 3 and norm(dt=9) == 3
    assert norm(w=None) == 1 and norm(r=A) == 1 and norm(c=A + 1) == 4
    gate = lambda x=A, dt=1, t=4, f=64, ld=128, fmt=1, c=A, s=A: lib.qo_swiglu_mx_quantize(_p(x), dt, t, f, ld, fmt, _p(c), _p(s), 2, _p(None))  # noqa: E731
    assert gate(t=0) == 0 and gate(ld=127) == 2 and gate(dt=3) == 3 and gate(x=None) == 1 and gate(c=A + 4) == 4
    gemm = lambda a=A, lda=32, fa=0, sa=A, sal=2, b=A, ldb=32, sb=A, sbl=2, bias=None, o=A, od=2, ldc=8, M=4, N=8, K=64, ws=None: lib.qo_mx_gemm(  # noqa: E731
        _p(a), lda, fa, _p(sa), sal, _p(b), ldb, _p(sb), sbl, _p(bias), _p(o), od, ldc, M, N, K, _p(ws), 0, _p(None))
    assert gemm(M=0) == 0 and gemm(N=0) == 0
    assert gemm(K=65) == 2 and gemm(K=-32) == 2 and gemm(M=-1) == 2 and gemm(ldc=7) == 2 and gemm(lda=16) == 2 and gemm(ldb=16) == 2
    assert gemm(fa=1) == 2 and gemm(sal=1) == 2 and gemm(sbl=1) == 2      # FP8 rows are twice as long
    assert gemm(fa=2) == 3 and gemm(od=3) == 3
    assert gemm(a=None) == 1 and gemm(o=None) == 1 and gemm(sb=None) == 1
    # more than 16 rows: scale rows of 16-byte multiples
    assert gemm(M=17) == 4 and gemm(M=17, sal=16, sbl=8) == 4 and gemm(M=17, sal=16, sbl=16, sa=A + 8) == 4
    assert gemm(M=17, sal=16, sbl=16, ws=A + 8) == 4
    assert gemm(a=A + 8) == 4 and gemm(b=A + 1) == 4 and gemm(lda=40) == 4 and gemm(ldb=33) == 4


def test_fakes_give_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(6, 100, dtype=torch.bfloat16, device="cuda")
        ops = torch.ops.quant_ops
        codes, scales = ops.mx_quantize(x)
        assert codes.shape == (6, 64) and codes.dtype == torch.uint8 and scales.shape == (6, 4)
        codes8, scales8, h = ops.add_rms_norm_mx_quantize(x, x, x[0])
        assert codes8.shape == (6, 128) and codes8.dtype == torch.float8_e4m3fn and h.shape == x.shape
        assert ops.rms_norm_mx_quantize(x, x[0], 1e-6, "mxfp4")[0].shape == (6, 64)
        assert ops.swiglu_mx_quantize(x)[0].shape == (6, 64)
        assert ops.mx_dequantize(codes, scales, 100, torch.float16).shape == (6, 100)
        out = ops.mx_matmul(codes8, scales8, codes, scales)
        assert out.shape == (6, 6) and out.dtype == torch.bfloat16
