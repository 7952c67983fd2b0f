"""A paged key/value cache held in 4 bits: appending keys and values with the position
rotation, attention over the cache, and reading it back.

Each token's key and value of each KV head is one vector of D values (64, 96, 128, 192 or
256), quantized asymmetrically: with v clamped to +-65504, lo = fp16(min v), s = fp16((max v
- lo) / 15), codes c = (v - lo) / s rounded to nearest even and clamped to 0 .. 15 (s = 0:
0). It reads as lo + s c. A vector that holds a NaN or an infinity reads as NaN.

A cache (:class:`KV4Cache`, made by :func:`kv4_cache`) is three contiguous tensors of pages
of P tokens (a power of two from 16 to 4096); a token's slot is page * P + its place in the
page:

* k_codes: uint8 [pages, heads, P, D/2], byte j holding value 2j (low bits) and 2j + 1;
* v_codes: uint8 [pages, heads, P/16, D/2, 16], the same bytes, 16 tokens side by side;
* params: float16 [pages, 2, heads, P/16, 2, 16]: keys and values; s and lo; 16 tokens.

Whole pages are copied by indexing the three tensors; D/2 + 4 bytes a vector.

GPU tensors use the HIP kernels through ``torch.ops.quant_ops``; if the HIP library is not
loaded they raise. Host tensors run the formulas in PyTorch. All of it is for inference:
nothing carries a gradient. None of these functions has a counterpart in the reference.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from . import _loader

HEAD_DIMS = (64, 96, 128, 192, 256)
MAX_PAGE = 4096
MAX_LENGTH = 2 ** 31 - 4096   # tokens of a sequence
_MOST = 65504.0
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class KV4Cache(NamedTuple):
    """The tensors of a cache (layout above)."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    params: torch.Tensor

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]


def kv4_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> KV4Cache:
    """A cache of zeros."""
    _check(pages >= 0 and kv_heads >= 1, f"invalid sizes: pages {pages}, kv_heads {kv_heads}")
    _check_sizes(page_size, head_dim)
    return KV4Cache(torch.zeros(pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device),
                    torch.zeros(pages, kv_heads, page_size // 16, head_dim // 2, 16, dtype=torch.uint8, device=device),
                    torch.zeros(pages, 2, kv_heads, page_size // 16, 2, 16, dtype=torch.float16, device=device))


def _check(ok, message):
    """Host tensors are refused where the GPU operators refuse them."""
    if not ok:
        raise ValueError(message)


def _check_sizes(page_size, head_dim):
    _check(16 <= page_size <= MAX_PAGE and page_size & (page_size - 1) == 0,
           f"page_size must be a power of two from 16 to {MAX_PAGE}, got {page_size}")
    _check(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")


def _check_cache(cache, on):
    k, v, p = cache
    _check(all(t.device == on.device for t in cache), "the cache and the other tensors must be on one device")
    _check(k.dtype == torch.uint8 and v.dtype == torch.uint8 and p.dtype == torch.float16,
           "the cache's codes must be uint8 and its params float16")
    _check(k.dim() == 4, f"not a cache: {tuple(k.shape)}")
    pages, heads, size, half = k.shape
    _check_sizes(size, 2 * half)
    _check(heads > 0, "the cache has no heads")
    _check(v.shape == (pages, heads, size // 16, half, 16) and p.shape == (pages, 2, heads, size // 16, 2, 16),
           f"the parts of the cache do not match: {tuple(k.shape)}, {tuple(v.shape)}, {tuple(p.shape)}")
    _check(all(t.is_contiguous() for t in cache), "the cache must be contiguous")


def _check_heads(x, like, cache, name):
    _check(x.dtype in _FLOATS, f"{name} dtype must be float32, float16 or bfloat16, got {x.dtype}")
    _check(x.dim() == 3 and x.shape[2] == cache.head_dim, f"{name} must be [tokens, heads, {cache.head_dim}], got {tuple(x.shape)}")
    _check(x.dtype == like.dtype and x.device == like.device and x.shape[0] == like.shape[0],
           f"{name} must have the others' tokens, dtype and device")


def _check_index(x, dtype, shape, on, name):
    _check(x.dtype == dtype and x.device == on.device, f"{name} must be {dtype} on the others' device, got {x.dtype}")
    _check(tuple(x.shape) == shape, f"{name} must have the shape {shape}, got {tuple(x.shape)}")


# Each operator's overload, looked up once. A library built before them lacks them: the
# package imports with it all the same.
_OPS = ("kv4_append", "kv4_read", "kv4_attention")
_op = {name: getattr(torch.ops.quant_ops, name).default for name in _OPS
       if _loader.KERNELS_AVAILABLE and hasattr(torch.ops.quant_ops, name)}


def _gpu(name):
    _loader.require_kernels(name)
    if name not in _op:
        raise RuntimeError(f"{name}: the loaded library ({_loader.TORCH_LIB_PATH}) does not have it; "
                           "rebuild with python -m quant_ops_amd._build")
    return _op[name]


# ------------------------------------------------------------------ host forms
def _quantize_pytorch(v):
    """Codes [..., D] (uint8) and params [..., 2] of float32 vectors."""
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], 0.0, v).clamp(-_MOST, _MOST)
    lo = v.amin(-1).half()
    s = ((v.amax(-1).double() - lo.double()) / 15).float().clamp(min=0).half()
    # in float64: the borders between codes
    c = (v.double() - lo.double()[..., None]) / torch.where(s == 0, 1.0, s.double())[..., None]
    c = torch.where(s[..., None] == 0, 0.0, torch.round(c).clamp(0, 15)).to(torch.uint8)
    return c, torch.where(bad[..., None], float("nan"), torch.stack((s, lo), -1))


def _rotate_pytorch(x, cos, sin, interleaved):
    """float32 rows of x [T, H, D] rotated by the angles of cos, sin [T, rot / 2]."""
    rot = 2 * cos.shape[1]
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack((a, b), 3).flatten(2) if interleaved else torch.cat((a, b), 2)
    return torch.cat((turned, x[..., rot:]), 2).float()


@torch.no_grad()
def _values_pytorch(cache, page, place):
    """float32 keys and values [..., heads, D] at (page, place)."""
    def values(codes, which):
        nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
        par = cache.params[page, which, :, place // 16, :, place % 16].float()
        return par[..., 1:] + par[..., :1] * nib

    return (values(cache.k_codes[page, :, place], 0),
            values(cache.v_codes[page, :, place // 16, :, place % 16], 1))


@torch.no_grad()
def _append_pytorch(cache, k, v, slots, positions, cos, sin, q, interleaved):
    keys = k.float()
    turned = None
    if cos is not None:
        known = (positions >= 0) & (positions < cos.shape[0])
        at = torch.where(known, positions, 0)
        c, s = torch.where(known[:, None], cos[at], float("nan")), sin[at]
        keys = _rotate_pytorch(keys, c, s, interleaved)
        turned = None if q is None else _rotate_pytorch(q, c, s, interleaved).to(q.dtype)
    size = cache.page_size
    keep = (slots >= 0) & (slots < cache.k_codes.shape[0] * size)
    page, place = slots[keep] // size, slots[keep] % size
    for which, x in enumerate((keys, v.float())):
        c, par = _quantize_pytorch(x[keep])
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
        if which == 0:
            cache.k_codes[page, :, place] = codes
        else:
            cache.v_codes[page, :, place // 16, :, place % 16] = codes
        cache.params[page, which, :, place // 16, :, place % 16] = par
    return turned


@torch.no_grad()
def _attention_pytorch(q, cache, page_table, lengths, scale, q_starts, window):
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    size, group = cache.page_size, q.shape[1] // cache.k_codes.shape[1]
    total, batch = q.shape[0], len(lengths)
    starts = q_starts.tolist() if q_starts is not None else [i * (total // max(batch, 1)) for i in range(batch + 1)]
    for b, length in enumerate(lengths.tolist()):
        lo, hi = (min(max(i, 0), total) for i in (starts[b] if b else 0, starts[b + 1]))
        if hi <= lo:
            continue
        if length > min(page_table.shape[1] * size, MAX_LENGTH):
            out[lo:hi] = float("nan")
            continue
        length = max(length, 0)
        t = torch.arange(length, device=q.device)
        page = page_table[b].long()[t // size]
        known = (page >= 0) & (page < cache.k_codes.shape[0])
        if bool(known.any()):
            k, v = _values_pytorch(cache, torch.where(known, page, 0), t % size)
        else:
            k, v = (q.new_zeros(length, cache.k_codes.shape[1], q.shape[2], dtype=torch.float32) for _ in range(2))
        # [heads, length, D]
        k, v = (torch.where(known[:, None, None], x, float("nan")).repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
        pos = torch.arange(length - (hi - lo), length, device=q.device)[:, None]
        seen = t <= pos
        if window:
            seen &= t > pos - window
        score = torch.matmul(q[lo:hi].float().transpose(0, 1), k.transpose(1, 2).contiguous()) * scale
        # [heads, queries, length]; a masked token's NaN stays out of the products
        p = torch.softmax(score.masked_fill(~seen, float("-inf")), 2).masked_fill(~seen, 0.0)
        bad = ~torch.isfinite(v).all(2)                      # [heads, length]
        o = torch.matmul(p, torch.where(bad[..., None], 0.0, v))
        o = torch.where((bad[:, None] & seen).any(2)[..., None], float("nan"), o)
        out[lo:hi] = o.transpose(0, 1).to(q.dtype)
    return out


# ------------------------------------------------------------------- operators
def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               interleaved: bool = False) -> Optional[torch.Tensor]:
    """Quantize k (rotated) and v [T, kv_heads, D] into the cache at slots [T] (int64), in place;
    the rotated q [T, q_heads, D], where one is given, is returned in its dtype.

    Slots outside the cache (-1 for padding) leave their token out; the others must differ (of
    two tokens in one slot the cache may hold a mix). With positions [T] (int64) and cos, sin
    (float32 [positions, rot / 2], rot a multiple of 8 up to D) the first rot values turn by
    their position's angles in pairs (i, i + rot / 2), or (2i, 2i + 1) if interleaved: (a, b) to (a cos
    - b sin, b cos + a sin), rounded to float32. A position outside the table gives NaN.
    k, v and q may be views of one projection's rows (any strides).
    """
    if k.is_cuda:
        out = _gpu("kv4_append")(cache.k_codes, cache.v_codes, cache.params, k, v, slots, positions, cos, sin, q, interleaved)
        return out if q is not None else None
    _check_cache(cache, k)
    tokens = k.shape[0]
    for x, name in ((k, "k"), (v, "v")) + (((q, "q"),) if q is not None else ()):
        _check_heads(x, k, cache, name)
    _check(k.shape[1] == v.shape[1] == cache.k_codes.shape[1], f"k and v must have the cache's {cache.k_codes.shape[1]} heads")
    _check_index(slots, torch.int64, (tokens,), k, "slots")
    _check((positions is None) == (cos is None) == (sin is None), "positions, cos and sin are given together or not at all")
    _check(q is None or cos is not None, "q is only rotated: it needs positions, cos and sin")
    if cos is not None:
        _check_index(positions, torch.int64, (tokens,), k, "positions")
        _check(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32 and cos.device == sin.device == k.device,
               "cos and sin must be float32 [positions, rot / 2] on the others' device")
        _check(cos.shape[0] > 0 and 0 < 2 * cos.shape[1] <= cache.head_dim and cos.shape[1] % 4 == 0,
               f"cos and sin {tuple(cos.shape)} must have rows of a multiple of 4 angles, {cache.head_dim // 2} at most")
    return _append_pytorch(cache, k, v, slots, positions, cos, sin, q, interleaved)


def kv4_read(cache: KV4Cache, slots: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [T, kv_heads, D] at slots [T] (int64): lo + s c in float32, rounded to
    out_dtype (float16: within +-65504); zeros for slots outside the cache."""
    if slots.is_cuda:
        return _gpu("kv4_read")(cache.k_codes, cache.v_codes, cache.params, slots, out_dtype)
    _check_cache(cache, slots)
    _check(slots.dim() == 1, f"slots must be 1-D, got {tuple(slots.shape)}")
    _check_index(slots, torch.int64, (slots.shape[0],), slots, "slots")
    _check(out_dtype in _FLOATS, f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    size = cache.page_size
    keep = (slots >= 0) & (slots < cache.k_codes.shape[0] * size)
    got = []
    for x in _values_pytorch(cache, slots[keep] // size, slots[keep] % size):
        out = torch.zeros(len(slots), *x.shape[1:], dtype=out_dtype, device=slots.device)
        out[keep] = (x.clamp(-_MOST, _MOST) if out_dtype == torch.float16 else x).to(out_dtype)
        got.append(out)
    return got[0], got[1]


def kv4_attention(q: torch.Tensor, cache: KV4Cache, page_table: torch.Tensor, lengths: torch.Tensor,
                  scale: Optional[float] = None, q_starts: Optional[torch.Tensor] = None, window: int = 0) -> torch.Tensor:
    """Causal attention of q [T, q_heads, D] over the cached keys and values: softmax(scale q k^T) v
    with float32 sums, in q's dtype. Query head h reads KV head h / (q_heads / kv_heads).

    page_table [B, W] (int32) holds the pages of each sequence in order, lengths [B] (int32)
    the sequences' cached tokens, those of the queries included. Sequence b has the queries q_starts[b]
    .. q_starts[b + 1] - 1 (int32 [B + 1], ascending from 0; rows from the last entry on give
    zeros), without q_starts T / B each. Query i of n of a sequence of L tokens stands at p = L - n
    + i and sees the tokens up to p, of a window those above p - window; zeros if there are none.
    scale (positive) defaults to 1 / sqrt(D).

    A query that sees a token on a page outside the cache gives NaN, and so do those of a sequence
    longer than its row of page_table or than 2^31 - 4096 tokens (entries past a sequence's tokens are not used). A narrower
    view of page_table tells the operator that no sequence is longer.
    """
    if scale is None:
        scale = cache.head_dim ** -0.5
    if q.is_cuda:
        return _gpu("kv4_attention")(q, cache.k_codes, cache.v_codes, cache.params, page_table, lengths, scale, q_starts, window)
    _check_cache(cache, q)
    _check_heads(q, q, cache, "q")
    _check(q.shape[1] > 0 and q.shape[1] % cache.k_codes.shape[1] == 0,
           f"q's heads ({q.shape[1]}) must be a multiple of the cache's {cache.k_codes.shape[1]}")
    _check(page_table.dim() == 2, f"page_table must be [sequences, pages], got {tuple(page_table.shape)}")
    batch = page_table.shape[0]
    _check_index(page_table, torch.int32, tuple(page_table.shape), q, "page_table")
    _check_index(lengths, torch.int32, (batch,), q, "lengths")
    if q_starts is not None:
        _check_index(q_starts, torch.int32, (batch + 1,), q, "q_starts")
    else:
        _check(q.shape[0] % batch == 0 if batch else q.shape[0] == 0, f"{q.shape[0]} queries of {batch} sequences need q_starts")
    _check(0 < scale < 3.4e38 and window >= 0, f"scale must be positive and window not negative, got {scale} and {window}")
    return _attention_pytorch(q, cache, page_table, lengths, scale, q_starts, window)
