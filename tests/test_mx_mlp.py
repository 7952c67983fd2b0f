"""The gated MLP of examples/mx_mlp.py against the block in float32.

Rounding e2m1 codes to a block's power of two gives a relative error of about 0.12 of a
normal tensor (e4m3 0.026), which normal errors of three products add as roots of squares:
the weights alone (mxfp8 activations) sqrt(3) * 0.12 = 0.21 at most, since gate and up share
their effect, with mxfp4 activations sqrt(2) times as much. The bound is a third above."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import mx_mlp  # noqa: E402

BOUND = {"mxfp8": 0.28, "mxfp4": 0.40}


def _check(tokens, features, hidden, fmt, device):
    weights, (x, residual) = mx_mlp.make(tokens, features, hidden, device, seed=tokens)
    out, h = mx_mlp.MXMLP(*weights, fmt=fmt)(x, residual)
    want, sums = mx_mlp.float_mlp(*weights, x, residual)
    assert out.shape == x.shape and out.dtype == x.dtype
    assert torch.equal(h, sums.to(x.dtype))
    assert mx_mlp.relative_error(out, want) < BOUND[fmt]


@pytest.mark.parametrize("fmt", ("mxfp8", "mxfp4"))
def test_block_on_the_host(fmt):
    _check(5, 256, 608, fmt, "cpu")


def test_command_on_the_host(capsys):
    assert mx_mlp.main(["--tokens", "3", "--features", "128", "--hidden", "320", "--device", "cpu"]) < BOUND["mxfp8"]
    assert "relative error" in capsys.readouterr().out


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ("mxfp8", "mxfp4"))
@pytest.mark.parametrize("tokens,features,hidden", [(1, 4096, 14336), (16, 1024, 2816), (100, 1000, 2720), (700, 4096, 1024)])
def test_block(gpu, tokens, features, hidden, fmt):
    print(f"[gpu-mx-mlp] {tokens} x {features} x {hidden} {fmt}", flush=True)
    _check(tokens, features, hidden, fmt, gpu)


@pytest.mark.gpu
def test_command(gpu, capsys):
    assert mx_mlp.main(["--tokens", "16", "--features", "1024", "--hidden", "2048"]) < BOUND["mxfp8"]
    assert "us replayed" in capsys.readouterr().out
