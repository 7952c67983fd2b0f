"""Attention over the 4-bit cache on the host: a sequence longer than the operators take is refused by its outputs, as on the
GPU, before anything of its length is made."""
import torch

import quant_ops_amd as qo


def test_longest_sequence():
    cache = qo.kv4_cache(1, 4096, 1, 64, device="cpu")
    table = torch.zeros(1, 1, dtype=torch.int32).expand(1, 2 ** 19)
    q = torch.ones(2, 1, 64)
    got = qo.kv4_attention(q, cache, table, torch.tensor([2 ** 31 - 4095], dtype=torch.int32))
    assert bool(torch.isnan(got).all())
