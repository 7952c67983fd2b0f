"""The operators of the 4-bit cache carry no gradient, on the host and on the GPU: inputs that require one leave the
cache and the results without a graph."""
import pytest
import torch

import quant_ops_amd as qo


def _step(device):
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(0)).to(device).requires_grad_()
    cos = torch.ones(4, 32, device=device).requires_grad_()
    cache = qo.kv4_cache(1, 16, 2, 64, device=device)
    slots = torch.arange(3, device=device)
    q = qo.kv4_append(cache, x, x, slots, positions=slots, cos=cos, sin=cos, q=x)
    k, v = qo.kv4_read(cache, slots)
    i32 = dict(dtype=torch.int32, device=device)
    out = qo.kv4_attention(x, cache, torch.zeros(3, 1, **i32), torch.tensor([1, 2, 3], **i32))
    return (q, k, v, out, *cache)


def _check(device):
    for t in _step(device):
        assert not t.requires_grad and t.grad_fn is None


def test_host():
    _check("cpu")


@pytest.mark.gpu
def test_gpu(gpu):
    _check(gpu)
