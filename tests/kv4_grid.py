"""Inputs of attention over the 4-bit cache whose scores float32 holds."""
import torch

from test_kv4_cpu import make


def on_a_grid(case, q_most):
    """Queries in eighths up to q_most and keys in sixteenths: scores below 2^16 in steps of 2^-7, which float32 holds and a
    product's sums reach without a rounding, so that two of a row are equal or 2^-7 apart."""
    q, cache, table, lengths, _, window = make(case, torch.float32)
    q = (q.clamp(-q_most, q_most) * 8).round() / 8
    cache.params[:, 0] = (cache.params[:, 0].float() * 16).round().half() / 16
    return q, cache, table, lengths, window
