"""Attention over a paged cache where numbers are large, against the formula in 64 bits."""

import pytest
import torch

from miles_amd.kernels.paged_attention import paged_attention
from miles_amd.kernels.paged_cache import PagedCache
from tests.operator_checks import f64, within
from tests.serving_checks import DEV

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]
PAGE = 16


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
