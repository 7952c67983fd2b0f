"""Caches, sequences and tolerances shared by the tests of the 4-bit key/value cache."""
import torch

import quant_ops_amd as qo
from oracle import kv4_reference as ok


def vectors(g, *shape):
    """N(0, 1) vectors of very different sizes and offsets, some constant."""
    x = torch.randn(*shape, generator=g)
    x = x * torch.exp2(torch.randint(-4, 4, (*shape[:-1], 1), generator=g).float())
    x = x + torch.randint(-2, 3, (*shape[:-1], 1), generator=g)
    if x.numel():
        x.view(-1, shape[-1])[::17] = 0.75
    return x


def angles(rows, rot):
    a = torch.arange(rows).double()[:, None] * 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
    return a.cos().float(), a.sin().float()


def random_cache(g, pages, page, heads, dim, size=1.0):
    """A cache of random codes and parameters (CPU), a few scales 0."""
    c = qo.kv4_cache(pages, page, heads, dim, device="cpu")
    c.k_codes.copy_(torch.randint(0, 256, c.k_codes.shape, generator=g))
    c.v_codes.copy_(torch.randint(0, 256, c.v_codes.shape, generator=g))
    s = size * (0.05 + 0.3 * torch.rand(c.params[:, :, :, :, 0].shape, generator=g))
    s[torch.rand(s.shape, generator=g) < 0.02] = 0.0
    c.params[:, :, :, :, 0] = s
    c.params[:, :, :, :, 1] = -7.5 * s + size * 0.3 * torch.randn(s.shape, generator=g)
    return c


def batch(g, lengths, page, spare=3):
    """A page table with every sequence's pages all over the cache, -1 behind them; the number of pages."""
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def bound(q, out, mag, big, lengths):
    """What the kernel's roundings may add up to, from the oracle's outputs, the magnitudes of their terms
    and of their scores'.

    A matrix product of codes is off by 2^-20 of its terms' magnitudes at most where they are subnormal
    (keys, 16-bit queries) and 2^-22 elsewhere (the largest measured on random operands is 7.5e-7 and
    1.9e-7), a float32 query by 2^-22 in its two fp16 parts; a score takes two more float32 roundings and
    the exponent's argument two, the exponential one. d, of a weight, counts in numerator and denominator.
    A weight's rounding to fp16 is half a step, 2^-11 (2^-22 in two parts). Sums over a lane's 16 tokens a
    step, over steps, waves and parts: a float32 rounding each. The division and the output's rounding."""
    few = q.dtype != torch.float32
    product = 2.0 ** -20 if few else 2.0 ** -22
    d = big * (product + (0 if few else 2.0 ** -22) + 2 * U) + 2 * big * 2 * U + 2 * U
    steps = max(lengths) / 64 + 16 + 70
    weight = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -22
    rel = 2 * d[..., None] + weight + 2.0 ** -22 + 2 * steps * U
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0   # half a subnormal step
    return (HALF_STEP[q.dtype] + 2 * U) * (out.abs() + rel * mag) + rel * mag + tiny


def check(q, got, cache, table, lengths, scale, starts=None, window=0):
    out, mag, big = ok.attention(q, cache, table, lengths, scale, starts, window)
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    fine = ~torch.isnan(out)
    off = (got - out).abs()[fine] / (bound(q, out, mag, big, lengths.tolist() + [0])[fine] + 1e-300)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst} of the bound"
    return worst
