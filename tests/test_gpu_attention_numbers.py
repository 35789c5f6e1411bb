"""Attention over a paged cache where numbers are large, small or infinite, against the formula in 64 bits."""

import math

import pytest
import torch

from miles_amd.kernels.paged_attention import paged_attention
from miles_amd.kernels.paged_cache import PagedCache
from tests.operator_checks import f64, within
from tests.serving_checks import DEV

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]
PAGE = 16
# What a weight is off by as a sum of 16-bit numbers.  bf16: nothing, three of them hold all its bits.  fp16: what is left without the last bits is below 2^-10 of it and
# rounded to 2^-11 of itself; and, of the largest among the same 32 tokens, which is 2^15, half of fp16's smallest steps of 2^-24, or one of them where nothing is left
WEIGHT = {torch.bfloat16: 0.0, torch.float16: 2.0**-21}
SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0**-39}
# bf16: two parts may be the smallest number where nothing is left, 2^-133, of weights whose largest in the sequence is 1 at least
LEAST = {torch.bfloat16: 2.0**-132, torch.float16: 0.0}


def _cache_of(sequences, dtype):
    """(cache, pages, lengths) of sequences [(keys [tokens, heads, key_dim], values)], one page behind the other."""
    used = [-(-k.shape[0] // PAGE) for k, _ in sequences]
    k, v = sequences[0]
    cache = PagedCache.empty(sum(used) + 1, PAGE, k.shape[1], k.shape[2], v.shape[2], dtype=dtype, device=DEV)
    table = torch.full((len(sequences), max(1, *used, 1)), -1, dtype=torch.int32)
    first = 0
    for i, ((k, v), n) in enumerate(zip(sequences, used)):
        table[i, :n] = torch.arange(first, first + n)
        at = torch.arange(k.shape[0], device=DEV)
        page, place = first + at // PAGE, at % PAGE
        cache.keys[page, :, :, place] = k.to(DEV).to(dtype).view(*k.shape[:2], k.shape[2] // 8, 8)
        cache.values[page, :, place] = v.to(DEV).to(dtype)
        first += n
    return cache, table.to(DEV), torch.tensor([k.shape[0] for k, _ in sequences], dtype=torch.int32, device=DEV)


def _widened(table, tokens):
    """The same pages in a table for `tokens` tokens, which the work is shared out by."""
    return torch.nn.functional.pad(table, (0, max(0, tokens // PAGE - table.shape[1])), value=-1)


def formula(q, k, v, scale=None):
    """(out [heads, value_dim] in 64 bits, a bound on what comes before its rounding) of q [heads, key_dim], k [tokens, key heads, key_dim], v.

    A score is a sum of key_dim products in fp32, off by (key_dim + 4) 2^-23 of their magnitudes, and is rounded twice more (times the scale, less the
    maximum), with the maximum and the exponential 2^-22 (1 + |score| + |maximum|); sums of n tokens are off by (n / 32 + 64) 2^-23 of the magnitudes.  These are errors of
    each token's own weight and of the total.  What a weight loses as 16-bit numbers is WEIGHT of itself and SMALLEST of the largest weight of its 32 tokens, LEAST of the
    largest of all."""
    dtype = q.dtype
    q, k, v = f64(q), f64(k), f64(v)
    group, n = q.shape[0] // k.shape[1], k.shape[0]
    k, v = (t.repeat_interleave(group, 1).transpose(0, 1).contiguous() for t in (k, v))
    scale = 1 / math.sqrt(q.shape[1]) if scale is None else scale
    scores = torch.matmul(k, q[:, :, None])[:, :, 0] * scale
    size = torch.matmul(k.abs(), q.abs()[:, :, None])[:, :, 0] * abs(scale)
    top = scores.amax(1, keepdim=True)
    w = torch.exp(scores - top)
    w = w / w.sum(1, keepdim=True)
    off = (q.shape[1] + 4) * 2.0**-23 * size + 2.0**-22 * (1 + scores.abs() + top.abs())
    of_sums = (n / 32 + 64) * 2.0**-23
    padded = torch.nn.functional.pad(w, (0, -n % 32)).view(q.shape[0], -1, 32)
    beside = padded.amax(2, keepdim=True).expand_as(padded).reshape(q.shape[0], -1)[:, :n]
    apart = w * (off + WEIGHT[dtype] + of_sums) + SMALLEST[dtype] * beside + LEAST[dtype] * w.amax(1, keepdim=True)
    out = torch.matmul(w[:, None], v)[:, 0]
    of_total = (w * off).sum(1, keepdim=True) + of_sums
    return out, torch.matmul(apart[:, None], v.abs())[:, 0] + of_total * out.abs()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("shared", [False, True], ids=["whole", "shared"])
@pytest.mark.parametrize("n", [1, 30, 700])
def test_scores_that_have_no_fraction(n, shared, dtype):
    """Scores so large that 32 bits have no place for units: the largest takes all, and of those that are the same each has its share."""
    size = 60000.0 if dtype == torch.float16 else 3e12
    q = torch.full((1, 2, 64), size, dtype=dtype, device=DEV)
    q[0, 1] *= 0.8125                                      # (an odd number of the last place's units)
    k = torch.full((n, 1, 64), 0.3 * size, dtype=dtype, device=DEV)
    v = torch.randn((n, 1, 64), generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).to(dtype)
    for first, winners in ((n // 2, 1), (n // 3, max(1, n // 4))):
        keys = k.clone()
        keys[first:first + winners] = 0.9 * size
        cache, table, lengths = _cache_of([(keys, v)], dtype)
        table = _widened(table, 6000) if shared else table
        out = paged_attention(q, cache, table, lengths)
        want = f64(v[first:first + winners, 0]).mean(0).expand(2, 64)
        within(out[0], want, (winners / 32 + 64) * 2.0**-23 * f64(v[first:first + winners, 0]).abs().mean(0), f"{winners} of {n}")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("shared", [False, True], ids=["whole", "shared"])
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("gap", [8.0, 14.0, 16.0, 18.0, 22.0, 81.0])
def test_a_first_token_that_has_nearly_all_weight(gap, spread, shared, dtype):
    """Its value is 0, so that a result is made of the others' small weights: none of them may be lost, however small, outside of its own step of 32."""
    g = torch.Generator().manual_seed(int(gap))
    heads, kv_heads, dim = 8, 2, 64
    sequences = []
    for n in (40, 64, 300, 2000):
        k, v = torch.zeros(n, kv_heads, dim), 200 * (2 + torch.randn(n, kv_heads, dim, generator=g))
        k[:, :, 0] = spread * torch.randn(n, kv_heads, generator=g)
        k[0, :, 0] = gap
        v[0] = 0
        sequences.append((k, v))
    cache, table, lengths = _cache_of(sequences, dtype)
    q = torch.zeros(len(sequences), heads, dim, dtype=dtype, device=DEV)
    q[:, :, 0] = 8                                         # times 1 / sqrt(64): a score is the key's first element
    out = paged_attention(q, cache, _widened(table, 6000) if shared else table, lengths)
    for i, (k, v) in enumerate(sequences):
        want, off = formula(q[i], k.to(DEV).to(dtype), v.to(DEV).to(dtype))
        within(out[i], want, off, f"{k.shape[0]} tokens")


def _random(lengths, heads, kv_heads, key_dim, value_dim, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(dtype)  # noqa: E731
    return randn(len(lengths), heads, key_dim), [(randn(n, kv_heads, key_dim), randn(n, kv_heads, value_dim)) for n in lengths]


def _check(out, q, sequences, which=None):
    for i in range(len(sequences)) if which is None else which:
        k, v = sequences[i]
        if k.shape[0] == 0:
            assert (out[i] == 0).all()
            continue
        want, off = formula(q[i], k, v)
        far = ~torch.isfinite(want)
        assert torch.equal(torch.nan_to_num(f64(out[i])[far], 7.0), torch.nan_to_num(want[far], 7.0)), f"sequence {i} of {k.shape[0]} tokens"
        within(out[i].masked_fill(far, 0), want.masked_fill(far, 0), off.masked_fill(far, 0), f"sequence {i} of {k.shape[0]} tokens")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lengths,heads,kv_heads,key_dim,value_dim,width", [
    ([1, 2, 33, 100], 4, 2, 64, 64, 0), ([1, 2, 33, 600], 4, 2, 64, 64, 6000), ([40, 500], 20, 1, 128, 256, 0), ([9000, 3, 700], 40, 1, 256, 256, 0), ([9000, 20], 8, 2, 128, 128, 0),
    ([0] * 299 + [5000], 4, 2, 64, 256, 0)], ids=["whole", "shared", "wide", "many heads", "long", "many sequences"])
def test_infinite_values_that_are_seen(lengths, heads, kv_heads, key_dim, value_dim, width, dtype):
    """One infinity among the values of an element makes its result that infinity, two of different signs a NaN; the other elements do not notice.
    All scores are within e^12 of each other, so that every token has a weight."""
    q, sequences = _random(lengths, heads, kv_heads, key_dim, value_dim, dtype)
    for k, v in sequences:
        n = v.shape[0]
        if n == 0:
            continue
        v[0, :, 3], v[n - 1, :, 5], v[n // 2, :, value_dim - 1] = math.inf, -math.inf, math.inf
        v[0, :, 9], v[n - 1, :, 10] = math.inf, math.inf
        if n > 1:
            v[n - 1, :, 9] = -math.inf
    cache, table, n = _cache_of(sequences, dtype)
    _check(paged_attention(q, cache, _widened(table, width), n), q, sequences)


@pytest.mark.parametrize("lengths,heads,kv_heads,key_dim,value_dim", [([130007], 2, 1, 64, 64), ([130007], 5, 1, 64, 256), ([0] * 150 + [40001] + [0] * 149, 4, 1, 64, 64), (
    [3] * 9 + [40001] + [0] * 290, 4, 1, 64, 256)])
def test_a_row_of_more_than_64_parts_a_wavefront_of_the_join(lengths, heads, kv_heads, key_dim, value_dim):
    """About a thousand parts for four wavefronts of a workgroup, and some 300 for one wavefront."""
    q, sequences = _random(lengths, heads, kv_heads, key_dim, value_dim, torch.bfloat16)
    cache, table, n = _cache_of(sequences, torch.bfloat16)
    out = paged_attention(q, cache, table, n)
    _check(out, q, sequences)
    assert torch.equal(out, paged_attention(q, cache, table, n))
