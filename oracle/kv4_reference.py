"""The 4-bit key/value cache from its definition, in 64 bits (for tests; no counterpart in the
reference).

Written apart from the package: tokens one at a time, codes by comparison with the borders
between them, bytes by their index in the layout, attention one query at a time.
"""
import torch


def half(v):
    """float64 values rounded to float32 and then to fp16."""
    return v.float().half().double()


def store(v):
    """Codes [..., D] (int64), s and lo [...] (float64) of float32 vectors v."""
    v = v.double()
    bad = ~torch.isfinite(v).all(-1)
    u = torch.where(torch.isfinite(v), v, 0.0).clamp(-65504, 65504)
    lo = half(u.amin(-1))
    s = half(((u.amax(-1) - lo) / 15).clamp(min=0))
    border = (torch.arange(15, dtype=torch.float64) + 0.5) * s[..., None]            # between c and c + 1
    d = (u - lo[..., None])[..., None]
    above = (d > border[..., None, :]) | ((d == border[..., None, :]) & (torch.arange(15) % 2 == 1))
    c = torch.where((s == 0)[..., None], 0, above.sum(-1))
    c = torch.where(bad[..., None], 0, c)
    nan = torch.tensor(float("nan"), dtype=torch.float64)
    return c, torch.where(bad, nan, s), torch.where(bad, nan, lo)


def turn(x, positions, cos, sin, interleaved):
    """x [T, H, D] rotated, float64; rounding to float32 is left to the caller."""
    x = x.double().clone()
    rot = 2 * cos.shape[1]
    for t, p in enumerate(positions.tolist()):
        for i in range(rot // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            if 0 <= p < cos.shape[0]:
                c, s = float(cos[p, i]), float(sin[p, i])
            else:
                c = s = float("nan")
            xa, xb = x[t, :, a].clone(), x[t, :, b].clone()
            x[t, :, a], x[t, :, b] = xa * c - xb * s, xb * c + xa * s
    return x


def put(cache, which, slot, c, s, lo):
    """Writes one token's codes [H, D], s and lo [H] into the tensors of a (CPU) cache, byte by byte."""
    k, v, params = cache
    size = k.shape[2]
    page, place = divmod(slot, size)
    for j in range(c.shape[1] // 2):
        byte = (c[:, 2 * j] + 16 * c[:, 2 * j + 1]).to(torch.uint8)
        if which == 0:
            k[page, :, place, j] = byte
        else:
            v[page, :, place // 16, j, place % 16] = byte
    params[page, which, :, place // 16, 0, place % 16] = s.half()
    params[page, which, :, place // 16, 1, place % 16] = lo.half()


def values(cache, which, slots):
    """float64 values [T, H, D] of slots (a list), and the size of their parts: of lo + s c or of (lo + 8 s) +
    s (c - 8), whichever is larger."""
    k, v, params = (t.cpu() for t in cache)
    at = torch.tensor(slots, dtype=torch.int64)
    page, place = at // k.shape[2], at % k.shape[2]
    b = (k[page, :, place] if which == 0 else v[page, :, place // 16, :, place % 16]).long()
    c = torch.stack((b % 16, b // 16), 3).flatten(2).double()
    par = params[page, which, :, place // 16, :, place % 16].double()
    s, lo = par[..., :1], par[..., 1:]
    return lo + s * c, torch.maximum(lo.abs() + s * c, (lo + 8 * s).abs() + s * (c - 8).abs())


def read(cache, which, slot, dtype):
    """[H, D] of one slot, as read back."""
    x = values(cache, which, [slot])[0][0].float()
    return (x.clamp(-65504, 65504) if dtype == torch.float16 else x).to(dtype)


def attention(q, cache, page_table, lengths, scale, q_starts=None, window=0):
    """On the CPU, float64 [T, H, D]: outputs, sum_t p (size of the values' parts), and the largest of the scores'
    magnitudes scale * sum |q| (size of the key's parts) [T, H]."""
    q, page_table, lengths = q.cpu().double(), page_table.cpu(), lengths.cpu()
    cache = tuple(t.cpu() for t in cache)
    pages, heads, size, _ = cache[0].shape
    group = q.shape[1] // heads
    out, mag, big = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    batch = len(lengths)
    starts = [i * (q.shape[0] // max(batch, 1)) for i in range(batch + 1)] if q_starts is None else q_starts.tolist()
    for b in range(batch):
        n, length = starts[b + 1] - starts[b], max(int(lengths[b]), 0)
        if n == 0:
            continue
        if length > page_table.shape[1] * size:
            out[starts[b]:starts[b + 1]] = float("nan")
            continue
        first = max(0, length - n + 1 - window) if window else 0
        ids = [int(page_table[b, t // size]) for t in range(first, length)]
        known = torch.tensor([0 <= i < pages for i in ids], dtype=torch.bool)
        slots = [i * size + t % size if ok else 0 for i, t, ok in zip(ids, range(first, length), known.tolist())]
        kv, parts = [], []
        for which in (0, 1):
            x, y = values(cache, which, slots) if bool(known.any()) else (torch.zeros(len(slots), heads, q.shape[2], dtype=torch.float64),) * 2
            kv.append(torch.where(known[:, None, None], x, float("nan")).repeat_interleave(group, 1))
            parts.append(y.repeat_interleave(group, 1))
        for i in range(n):
            p = length - n + i
            lo, hi = max(0, p - window + 1) if window else 0, p + 1
            if hi <= lo:
                continue
            k, v = (x[lo - first:hi - first] for x in kv)   # [t, H, D]
            kp, vp = (x[lo - first:hi - first] for x in parts)
            w = torch.softmax((k * q[starts[b] + i]).sum(2) * scale, 0)
            out[starts[b] + i] = (w[..., None] * v).sum(0)
            mag[starts[b] + i] = (w[..., None] * vp).sum(0)
            big[starts[b] + i] = (kp * q[starts[b] + i].abs()).sum(2).amax(0) * scale
    return out, mag, big
