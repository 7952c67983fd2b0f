"""A transformer's gated MLP block with microscaled activations and 4-bit weights.

Four calls after the weights are prepared: RMS norm of the residual stream with
quantized output, gate and up product, SwiGLU with quantized output, down product.
No activation stands in memory between them in more than 8 bits but the gate and up
product's output.

    python examples/mx_mlp.py --tokens 16 --features 4096 --hidden 14336 --fmt mxfp8

prints the error against the same block in float32 with the weights as given, and on
a GPU the time of a call, eager and as a replayed graph.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import quant_ops_amd as qo  # noqa: E402


class MXMLP:
    """x, residual [..., F] -> (mlp(norm(x + residual)), x + residual).

    norm [F], gate and up [H, F], down [F, H]: the weights, kept as mxfp4 codes and
    scales; fmt: the activations' format.
    """

    def __init__(self, norm, gate, up, down, eps=1e-6, fmt="mxfp8"):
        self.norm, self.eps, self.fmt = norm, eps, fmt
        self.gate_up = qo.mx_quantize(torch.cat((gate, up)), "mxfp4")
        self.down = qo.mx_quantize(down, "mxfp4")

    def __call__(self, x, residual):
        codes, scales, h = qo.rms_norm_mx_quantize(x, self.norm, self.eps, residual=residual, fmt=self.fmt)
        gate_up = qo.mx_matmul(codes, scales, *self.gate_up, out_dtype=x.dtype)
        codes, scales = qo.swiglu_mx_quantize(gate_up, self.fmt)
        return qo.mx_matmul(codes, scales, *self.down, out_dtype=x.dtype), h


def float_mlp(norm, gate, up, down, x, residual, eps=1e-6):
    """The block in float32, nothing quantized."""
    norm, gate, up, down, h = (t.float() for t in (norm, gate, up, down, x.float() + residual.float()))
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * norm
    return (torch.nn.functional.silu(y @ gate.t()) * (y @ up.t())) @ down.t(), h


def make(tokens, features, hidden, device, dtype=torch.bfloat16, seed=0):
    """Weights (norm, gate, up, down) and inputs (x, residual)."""
    g = torch.Generator().manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g)).to(device, dtype)

    weights = (1 + randn(features, scale=0.1), randn(hidden, features, scale=features ** -0.5),
               randn(hidden, features, scale=features ** -0.5), randn(features, hidden, scale=hidden ** -0.5))
    return weights, (randn(tokens, features), randn(tokens, features))


def relative_error(got, want):
    return float((got.float() - want.float()).norm() / want.float().norm())


def _time(call, calls=50):
    for _ in range(5):
        call()
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(calls):
        call()
    torch.cuda.synchronize()
    return (time.perf_counter() - start) / calls * 1e6


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--tokens", type=int, default=16)
    p.add_argument("--features", type=int, default=4096)
    p.add_argument("--hidden", type=int, default=14336)
    p.add_argument("--fmt", choices=("mxfp4", "mxfp8"), default="mxfp8")
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    args = p.parse_args(argv)
    weights, (x, residual) = make(args.tokens, args.features, args.hidden, args.device)
    mlp = MXMLP(*weights, fmt=args.fmt)
    out, h = mlp(x, residual)
    want, _ = float_mlp(*weights, x, residual)
    error = relative_error(out, want)
    print(f"{args.tokens} x {args.features}, hidden {args.hidden}, {args.fmt}: relative error {error:.4f} against float32")
    if x.is_cuda:
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            mlp(x, residual)
        print(f"{_time(lambda: mlp(x, residual)):.1f} us a call, {_time(graph.replay):.1f} us replayed")
    return error


if __name__ == "__main__":
    main()
