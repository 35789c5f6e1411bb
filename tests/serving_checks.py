"""Rotary positions and attention over a paged cache in 64 bits, and how far a result may be from them."""

import math

import torch

from miles_amd.kernels.paged_cache import PagedCache
from tests.operator_checks import f64

DEV = "cuda:0"


def turned64(x, positions, inv_freq, scale=1.0, interleaved=False, back=False):
    """(the turned tensor, a bound on what 32-bit products and sums of 32-bit cosines and sines are off by)

    Cosine and sine are rounded once (2^-24 of themselves), so is each product and the sum: three roundings of a magnitude of at most
    |a c| + |b s|; the last factor covers the angle, whose 64 bits are far below."""
    x = f64(x)
    angle = positions.double()[..., None, None] * inv_freq.double()
    c, s = torch.cos(angle) * scale, torch.sin(angle) * (-scale if back else scale)
    n = inv_freq.shape[0]
    even, odd = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out, off = x.clone(), torch.zeros_like(x)
    a, b = x[..., even], x[..., odd]
    out[..., even], out[..., odd] = a * c - b * s, b * c + a * s
    off[..., even], off[..., odd] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, 3.01 * 2.0**-24 * off


def make_cache(pages, page_size, kv_heads, key_dim, value_dim, dtype, kept8=False, fill=None, generator=None):
    """A cache whose places hold random vectors, or `fill`."""
    cache = PagedCache.empty(pages, page_size, kv_heads, key_dim, value_dim, dtype=dtype, kept8=kept8, device=DEV)
    for t in (cache.keys, cache.values):
        if fill is not None:
            t.copy_(torch.full(t.shape, fill, dtype=torch.float32, device=DEV))
        else:
            t.copy_(torch.randn(t.shape, generator=generator, device=DEV))
    for t in (cache.key_scales, cache.value_scales):
        if t is not None and fill is not None:
            t.fill_(255)                                   # a NaN
        elif t is not None:
            t.copy_(torch.randint(119, 128, t.shape, generator=generator, device=DEV))
    return cache


def attend64(q, k, v, scale=None, sinks=None):
    """(out [heads, value_dim], a bound on what comes before its rounding), of one query [heads, key_dim] over k [tokens, kv heads, key_dim], v.

    The bound: a score is a sum of key_dim products in fp32, off by (key_dim + 4) 2^-23 of their magnitudes, and what an exponential's argument
    and value are rounded to is 2^-22 + 2^-22 of the score and the maximum; a weight is held in two 16-bit numbers, off by 2^-17 of itself or, for
    small fp16 ones, by 2^-25 of the largest; sums of n tokens, 32 at a time, are off by (n / 32 + 64) 2^-23 of the magnitudes."""
    q, k, v = f64(q), f64(k), f64(v)
    heads, n = q.shape[0], k.shape[0]
    if n == 0:
        return torch.zeros(heads, v.shape[2], dtype=torch.float64, device=q.device), torch.zeros(heads, v.shape[2], dtype=torch.float64, device=q.device)
    group = heads // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scale = 1 / math.sqrt(q.shape[1]) if scale is None else scale
    scores = torch.matmul(k.transpose(0, 1), q[:, :, None])[:, :, 0] * scale
    size = torch.matmul(k.abs().transpose(0, 1), q.abs()[:, :, None])[:, :, 0] * abs(scale)
    top = scores.amax(1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, f64(sinks)[:, None])
    p = torch.exp(scores - top)
    total = p.sum(1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(f64(sinks)[:, None] - top)
    w = p / total
    off = (q.shape[1] + 4) * 2.0**-23 * size + 2.0**-22 * (1 + scores.abs() + top.abs())
    share = 2 * off.amax(1) + 2.0**-17 + (n / 32 + 64) * 2.0**-23
    magnitude = torch.matmul(w[:, None], v.abs().transpose(0, 1))[:, 0]
    # (the rest of a weight that two fp16 numbers have no place for: relative to the largest weight of those that are summed)
    tiny = 2.0**-25 * v.abs().sum(0) / torch.exp(scores - scores.amax(1, keepdim=True)).sum(1)[:, None]
    return torch.matmul(w[:, None], v.transpose(0, 1))[:, 0], share[:, None] * magnitude + tiny
