"""Attention of one token a sequence over a paged cache, against the formula in 64 bits."""

import pytest
import torch

from miles_amd.kernels.paged_attention import paged_attention
from miles_amd.kernels.paged_cache import PagedCache
from tests.operator_checks import within
from tests.serving_checks import DEV, attend64, make_cache

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


def _setup(lengths, heads, kv_heads, key_dim, value_dim, page_size, dtype, kept8=False, width=None, seed=0):
    """(q, cache, pages, lengths): pages in any order, those behind a sequence's last one numbers that the cache has not."""
    g = torch.Generator().manual_seed(seed)
    used = [max(0, -(-n // page_size)) for n in lengths]
    width = max([1, *used]) if width is None else width
    total = sum(used) + 2
    order = torch.randperm(total, generator=g)
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n].int()
        at += n
    cache = make_cache(total, page_size, kv_heads, key_dim, value_dim, dtype, kept8, generator=torch.Generator(device=DEV).manual_seed(seed))
    q = (1.5 * torch.randn(len(lengths), heads, key_dim, generator=g)).to(dtype).to(DEV)
    return q, cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def _slots(cache, table, i, low, high):
    at = torch.arange(low, high, device=DEV)
    return table[i, at // cache.page_size].long() * cache.page_size + at % cache.page_size


def _check(out, q, cache, table, lengths, window=None, sinks=None, scale=None, which=None):
    for i in range(len(lengths)) if which is None else which:
        n = lengths[i].item()
        low = max(0, n - window) if window else 0
        if n <= 0:
            assert (out[i] == 0).all()
            continue
        k, v = cache.gather(_slots(cache, table, i, low, n), q.dtype)
        want, off = attend64(q[i], k, v, scale, sinks)
        within(out[i], want, off, f"sequence {i} of {n}")


# lengths around steps of 16 and 32 and pages; the table as wide as the longest needs, and so wide that the work is shared out by lengths
LENGTHS = [1, 0, 15, 16, 17, 31, 32, 33, 64, 0, 100, 127, 128, 129, 255, 300, 2]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("wide", [False, True], ids=["whole", "shared"])
@pytest.mark.parametrize("heads,kv_heads,key_dim,value_dim,page_size", [
    (1, 1, 64, 64, 16), (8, 2, 128, 128, 16), (32, 8, 128, 128, 64), (6, 2, 192, 128, 32), (5, 1, 256, 256, 16), (20, 1, 64, 128, 128), (40, 1, 128, 128, 256),
    (128, 1, 96, 160, 16), (34, 2, 32, 32, 1024), (48, 16, 160, 256, 32), (80, 1, 192, 192, 64)])
def test_attention(heads, kv_heads, key_dim, value_dim, page_size, wide, kept8, dtype):
    q, cache, table, lengths = _setup(LENGTHS, heads, kv_heads, key_dim, value_dim, page_size, dtype, kept8, width=-(-5000 // page_size) if wide else None, seed=heads)
    out = paged_attention(q, cache, table, lengths)
    assert out.shape == (len(LENGTHS), heads, value_dim) and out.dtype == dtype
    _check(out, q, cache, table, lengths)
    assert torch.equal(out, paged_attention(q, cache, table, lengths))


@pytest.mark.parametrize("key_dim,value_dim", [(8, 8), (72, 72), (80, 80), (112, 104), (200, 136), (248, 8), (16, 256)])
@pytest.mark.parametrize("wide", [False, True], ids=["whole", "shared"])
def test_odd_widths(key_dim, value_dim, wide):
    q, cache, table, lengths = _setup([1, 40, 333, 0, 16], 6, 2, key_dim, value_dim, 16, torch.bfloat16, width=400 if wide else None)
    _check(paged_attention(q, cache, table, lengths), q, cache, table, lengths)


@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page_size", [
    ([20000], 4, 1, 128, 16), ([5000, 1, 3, 7000, 0, 9], 8, 2, 128, 64), ([4096] * 3, 40, 1, 256, 32), ([9001, 33], 16, 16, 64, 16), ([1] * 40 + [6000] + [17] * 30, 8, 4, 128, 16)])
def test_long_sequences_are_shared_out(lengths, heads, kv_heads, dim, page_size, kept8):
    q, cache, table, n = _setup(lengths, heads, kv_heads, dim, dim, page_size, torch.bfloat16, kept8)
    out = paged_attention(q, cache, table, n)
    _check(out, q, cache, table, n)
    assert torch.equal(out, paged_attention(q, cache, table, n))


@pytest.mark.parametrize("batch", [255, 256, 257, 700, 1500])
def test_many_sequences(batch):
    """More sequences than the lanes of a workgroup, which add up the lengths."""
    lengths = [(i * 37) % 90 for i in range(batch)]
    q, cache, table, n = _setup(lengths, 4, 2, 64, 64, 16, torch.bfloat16, width=100)
    out = paged_attention(q, cache, table, n)
    _check(out, q, cache, table, n, which=range(0, batch, 7))
    assert (out[n == 0] == 0).all() and torch.isfinite(out).all()
    # the same sequences one behind the other, where none is shared: sums in another order
    alone = paged_attention(q, cache, table[:, :8].contiguous(), n)
    assert (out.float() - alone.float()).abs().max() <= 2.0**-6


@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("wide", [False, True], ids=["whole", "shared"])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 1000])
def test_windows_and_sinks(window, wide, kept8):
    q, cache, table, lengths = _setup([1, 16, 100, 333, 0, 1777], 12, 2, 64, 96, 16, torch.bfloat16, kept8, width=500 if wide else None)
    sinks = torch.randn(12, generator=torch.Generator().manual_seed(1)).to(DEV)
    sinks[3], sinks[4] = float("-inf"), 30.0
    for s in (None, sinks):
        _check(paged_attention(q, cache, table, lengths, window=window, sinks=s), q, cache, table, lengths, window, s)
    # pages before the window are anybody's: numbers that the cache has not
    gone = table.clone()
    for i, n in enumerate(lengths.tolist()):
        gone[i, :max(0, n - window) // 16] = 1 << 30
    assert torch.equal(paged_attention(q, cache, gone, lengths, window=window, sinks=sinks), paged_attention(q, cache, table, lengths, window=window, sinks=sinks))


@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0])
def test_scales(scale):
    q, cache, table, lengths = _setup([77, 1000], 4, 2, 64, 64, 16, torch.float16)
    _check(paged_attention(q, cache, table, lengths, scale=scale), q, cache, table, lengths, scale=scale)


@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("wide", [False, True], ids=["whole", "shared"])
@pytest.mark.parametrize("window", [None, 21])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf")])
def test_what_lies_in_places_that_are_not_seen_does_not_matter(garbage, window, wide, kept8):
    """A cache of NaNs (in 8 bits their scales are NaNs as well) with finite vectors in the places that are seen alone."""
    q, cache, table, lengths = _setup([1, 37, 64, 0, 250, 16], 8, 2, 128, 64, 32, torch.bfloat16, kept8, width=200 if wide else None)
    want = paged_attention(q, cache, table, lengths, window=window)
    spoilt = make_cache(cache.pages, 32, 2, 128, 64, torch.bfloat16, kept8, fill=garbage)
    for i, n in enumerate(lengths.tolist()):
        slots = _slots(cache, table, i, max(0, n - window) if window else 0, n)
        page, place = slots // 32, slots % 32
        for name in ("keys", "values", "key_scales", "value_scales"):
            to, of = getattr(spoilt, name), getattr(cache, name)
            if to is None:
                continue
            to, of = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (to, of))
            if name == "values":
                to[page, :, place] = of[page, :, place]
            else:
                to[page, :, :, place] = of[page, :, :, place]
    assert torch.equal(paged_attention(q, spoilt, table, lengths, window=window), want)


@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("wide", [False, True], ids=["whole", "shared"])
def test_pages_that_the_cache_has_not_are_left_out(wide, kept8):
    lengths = [100, 40, 16, 200]
    q, cache, table, n = _setup(lengths, 4, 2, 64, 64, 16, torch.bfloat16, kept8, width=300 if wide else None)
    bad = [(0, 2), (1, 0), (2, 0), (3, 12), (3, 5)]
    for (i, page), number in zip(bad, (-1, cache.pages, 2**31 - 1, -(2**31), cache.pages + 5)):
        table[i, page] = number
    out = paged_attention(q, cache, table, n)
    for i, length in enumerate(lengths):
        slots = _slots(cache, table, i, 0, length)
        k, v = cache.gather(slots[(slots >= 0) & (slots < cache.pages * 16)], q.dtype)
        want, off = attend64(q[i], k, v)
        within(out[i], want, off, f"sequence {i}")
    assert (out[2] == 0).all()


def test_lengths_beyond_the_table_and_below_zero():
    q, cache, table, n = _setup([64, 64, 64], 4, 2, 64, 64, 16, torch.bfloat16)
    want = paged_attention(q, cache, table, n)
    out = paged_attention(q, cache, table, torch.tensor([65, 2**31 - 1, -3], dtype=torch.int32, device=DEV))
    assert torch.equal(out[:2], want[:2]) and (out[2] == 0).all()
    assert (paged_attention(q, cache, table[:, :0], n) == 0).all()
    assert paged_attention(q[:0], cache, table[:0], n[:0]).shape == (0, 4, 64)


def test_inputs_of_other_places_and_orders():
    q, cache, table, n = _setup([64, 700, 3], 8, 2, 64, 64, 16, torch.bfloat16)
    want = paged_attention(q, cache, table, n)
    fused = torch.zeros(3, 10, 64, dtype=q.dtype, device=DEV)
    fused[:, 1:9] = q
    off = torch.nn.functional.pad(q, (3, 2))[..., 3:-2]
    for other in (fused[:, 1:9], off, q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(paged_attention(other, cache, table, n), want)
    wide = torch.full((3, 60), -1, dtype=torch.int32, device=DEV)
    wide[:, 5:5 + table.shape[1]] = table
    for other in (wide[:, 5:5 + table.shape[1]], table.t().contiguous().t()):
        assert torch.equal(paged_attention(q, cache, other, n), want)
    assert torch.equal(paged_attention(q[:1].expand(3, 8, 64), cache, table[:1].expand(3, -1), n[:1].expand(3)), paged_attention(q[:1], cache, table[:1], n[:1]).expand(3, 8, 64))


def test_scores_far_apart_and_all_alike():
    """One token that outweighs all others by far, tokens of equal weight, scores beyond the exponential's range."""
    q, cache, table, n = _setup([500], 4, 1, 64, 64, 16, torch.float16)
    slots = _slots(cache, table, 0, 0, 500)
    cache.keys.zero_()
    out = paged_attention(q, cache, table, n)
    _check(out, q, cache, table, n)
    page, place = slots[313] // 16, slots[313] % 16
    for size in (4.0, 200.0, 60000.0):
        cache.keys[page, 0, :, place] = (q[0, 1].float() * size / q[0, 1].float().abs().max()).half().view(8, 8)
        _check(paged_attention(q, cache, table, n), q, cache, table, n)
        _check(paged_attention(-q, cache, table, n), -q, cache, table, n)


def test_a_cache_beyond_32_bits():
    pages = 5 * (1 << 30) // 2 // (64 * 8 * 128 * 2) + 1
    cache = PagedCache.empty(pages, 64, 8, 128, 128, device=DEV)
    table = torch.tensor([[pages - 1, 0, pages - 2], [pages // 2, pages - 3, 1]], dtype=torch.int32, device=DEV)
    for p in table.flatten().tolist():
        cache.keys[p].normal_(), cache.values[p].normal_()
    q = torch.randn(2, 32, 128, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    n = torch.tensor([190, 129], dtype=torch.int32, device=DEV)
    _check(paged_attention(q, cache, table, n), q, cache, table, n)


def test_refusals():
    q, cache, table, n = _setup([20, 20], 4, 2, 64, 64, 16, torch.bfloat16)
    sinks = torch.zeros(4, device=DEV)
    for args, kw, text in (((q[:, :3], cache, table, n), {}, "q of shape"), ((q[..., :32], cache, table, n), {}, "q of shape"), ((q.half(), cache, table, n), {}, "a cache of"),
                           ((q, cache, table[:1], n), {}, "pages of shape"), ((q, cache, table, n[:1]), {}, "lengths of shape"), ((q, cache, table.long(), n), {}, "int32"),
                           ((q, cache, table, n.long()), {}, "int32"), ((q, cache, table.cpu(), n), {}, "pages on"), ((q, cache, table, n), dict(sinks=sinks[:3]), "sinks are"),
                           ((q, cache, table, n), dict(sinks=sinks.half()), "sinks are"), ((q, cache, table, n), dict(window=0), "window"),
                           ((q.clone().requires_grad_(True), cache, table, n), {}, "no_grad"), ((q.float(), cache, table, n), {}, "bfloat16 or float16")):
        with pytest.raises(ValueError, match=text):
            paged_attention(*args, **kw)
