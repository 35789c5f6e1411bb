"""Tokens appended to a paged cache: what lies in their slots, and that nothing else is touched."""

import pytest
import torch

from miles_amd.kernels.paged_cache import PagedCache, append_tokens
from miles_amd.kernels.rotary import rotary, rotary_frequencies
from miles_amd.utils.mxfp8 import mxfp8_quantize
from tests.serving_checks import DEV, make_cache

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


def _raw(cache):
    return [t.view(torch.uint8) for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales) if t is not None]


def _inputs(tokens, heads, kv_heads, key_dim, value_dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    fused = (torch.randn(tokens, (heads + kv_heads) * key_dim + kv_heads * value_dim, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g))).to(dtype).to(DEV)
    q, k, v = fused.split((heads * key_dim, kv_heads * key_dim, kv_heads * value_dim), 1)
    return q.unflatten(1, (heads, key_dim)), k.unflatten(1, (kv_heads, key_dim)), v.unflatten(1, (kv_heads, value_dim))


def _slots(tokens, count, seed=0):
    """Different slots in any order; every fifth token has none."""
    slots = torch.randperm(count, generator=torch.Generator().manual_seed(seed))[:tokens]
    outside = torch.tensor([-1, count, -(1 << 40), count + (1 << 33)])
    slots[4::5] = outside[torch.arange(len(slots[4::5])) % 4]
    return slots.to(DEV)


def _rows(cache, slots):
    """The raw contents of slots: keys [n, heads, key_dim], values, scales of both, as the cache's layout has them."""
    page, place = slots // cache.page_size, slots % cache.page_size
    out = [cache.keys.view(torch.uint8)[page, :, :, place].flatten(2), cache.values.view(torch.uint8)[page, :, place]]
    return out + [t[page, :, :, place] for t in (cache.key_scales, cache.value_scales) if t is not None]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("tokens,kv_heads,key_dim,value_dim,page_size,pairs,interleaved", [
    (1, 1, 64, 64, 16, 32, False), (7, 2, 128, 128, 16, 64, False), (100, 3, 192, 128, 64, 32, True), (2000, 8, 128, 128, 16, 64, False), (4099, 1, 256, 256, 128, 64, False),
    (33, 5, 96, 32, 32, 48, False), (50, 2, 32, 160, 256, 16, True), (64, 4, 128, 64, 1024, 0, False), (9000, 2, 64, 96, 32, 8, True), (3, 16, 256, 32, 16, 24, False)])
def test_appended(tokens, kv_heads, key_dim, value_dim, page_size, pairs, interleaved, kept8, dtype):
    q, k, v = _inputs(tokens, 3 * kv_heads, kv_heads, key_dim, value_dim, dtype, seed=tokens)
    pages = (tokens + 3 * page_size) // page_size + 2
    cache = make_cache(pages, page_size, kv_heads, key_dim, value_dim, dtype, kept8, generator=torch.Generator(device=DEV).manual_seed(1))
    before = [t.clone() for t in _raw(cache)]
    slots = _slots(tokens, pages * page_size, seed=tokens)
    kw, turned_k = {}, k
    if pairs:
        freq, positions = rotary_frequencies(2 * pairs, device=DEV)[0], torch.arange(tokens, device=DEV) * 31 + 5
        kw = dict(positions=positions, inv_freq=freq, interleaved=interleaved, scale=1.125, q=q)
        turn = lambda t: rotary(t, None, positions, freq, interleaved=interleaved, scale=1.125)  # noqa: E731
        turned_k = turn(k.float() if kept8 else k)
    out = append_tokens(cache, k, v, slots, **kw)
    assert torch.equal(out, turn(q)) if pairs else out is None
    inside = (slots >= 0) & (slots < pages * page_size)
    rows = _rows(cache, slots[inside])
    for i, t in enumerate((turned_k, v)):
        if kept8:
            codes, scales = mxfp8_quantize(t[inside].reshape(-1, t.shape[-1]).contiguous())
            assert torch.equal(rows[i].reshape(codes.shape), codes.view(torch.uint8)) and torch.equal(rows[2 + i].reshape(scales.shape), scales)
        else:
            assert torch.equal(rows[i].contiguous().view(dtype), t[inside])
    # what the cache itself says lies there
    got_k, got_v = cache.gather(slots[inside], dtype)
    assert got_k.shape == k[inside].shape and got_v.shape == v[inside].shape
    if not kept8:
        assert torch.equal(got_k, turned_k[inside]) and torch.equal(got_v, v[inside])
    # every other place as it was
    restore = PagedCache(cache.keys.clone(), cache.values.clone(), *(None if t is None else t.clone() for t in (cache.key_scales, cache.value_scales)))
    page, place = slots[inside] // page_size, slots[inside] % page_size
    for nth, (t, b) in enumerate(zip(_raw(restore), before)):
        if nth == 1:                                       # values: places before elements
            t[page, :, place] = b[page, :, place]
        else:
            t[page, :, :, place] = b[page, :, :, place]
    assert all(torch.equal(t, b) for t, b in zip(_raw(restore), before))


@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
def test_inputs_of_other_places_and_types(kept8):
    """Addresses that are no multiples of 16, other orders, int32 slots and positions, expanded tensors."""
    q, k, v = (t.contiguous() for t in _inputs(40, 4, 2, 64, 96, torch.bfloat16))
    freq, positions, slots = rotary_frequencies(64, device=DEV)[0], torch.arange(40, device=DEV), _slots(40, 64)
    want = make_cache(4, 16, 2, 64, 96, torch.bfloat16, kept8, fill=1.0)
    out = append_tokens(want, k, v, slots, positions=positions, inv_freq=freq, q=q)
    off = lambda t: torch.nn.functional.pad(t, (3, 2))[..., 3:-2]  # noqa: E731
    small = torch.where(slots.abs() < 1 << 20, slots, -1).int()
    for a, b, c in ((off(q), off(k), off(v)), (q.transpose(0, 1).contiguous().transpose(0, 1),) * 1 + (k.flip(0).flip(0), v.transpose(1, 2).contiguous().transpose(1, 2))):
        cache = make_cache(4, 16, 2, 64, 96, torch.bfloat16, kept8, fill=1.0)
        got = append_tokens(cache, b, c, small, positions=positions.int(), inv_freq=freq, q=a)
        assert torch.equal(got, out) and all(torch.equal(x, y) for x, y in zip(_raw(cache), _raw(want)))
    one = append_tokens(cache, k[:1].expand(40, 2, 64), v[:1].expand(40, 2, 96), slots, positions=positions[:1], inv_freq=freq.float(), q=q[:1].expand(40, 4, 64))
    assert torch.equal(one, one[:1].expand_as(one))
    assert append_tokens(cache, k[:0], v[:0], slots[:0]) is None


def test_a_slot_that_is_given_twice_and_infinite_values():
    q, k, v = (t.contiguous() for t in _inputs(3, 2, 1, 64, 64, torch.bfloat16))
    cache = make_cache(2, 16, 1, 64, 64, torch.bfloat16, fill=5.0)
    append_tokens(cache, k, v, torch.tensor([3, 3, 9], device=DEV))
    got, _ = cache.gather(torch.tensor([3, 9], device=DEV))
    assert ((got[0] == k[0]) | (got[0] == k[1])).all() and torch.equal(got[1], k[2])
    others = torch.tensor([s for s in range(32) if s not in (3, 9)], device=DEV)
    assert (cache.gather(others)[0] == 5).all() and (cache.gather(others)[1] == 5).all()
    cache = make_cache(2, 16, 1, 64, 64, torch.bfloat16, kept8=True, fill=1.0)
    v[0, 0, 7], v[1, 0, 40], v[2] = float("inf"), float("nan"), 0
    append_tokens(cache, k, v, torch.tensor([0, 1, 2], device=DEV))
    codes, scales = mxfp8_quantize(v.reshape(3, 64))
    rows = _rows(cache, torch.arange(3, device=DEV))
    got, want = rows[1].reshape(3, 64).view(torch.float8_e4m3fn).float(), codes.float()      # (a NaN of either sign is one)
    assert torch.equal(got.isnan(), want.isnan()) and want.isnan().sum() == 1 and torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    assert torch.equal(rows[3].reshape(3, 2), scales)


def test_a_cache_beyond_32_bits():
    """Five GiB of pages: offsets of its last ones in bytes and in elements have no 32 bits."""
    pages, heads, dim = 5 * (1 << 30) // 2 // (64 * 8 * 128 * 2) + 1, 8, 128
    cache = PagedCache.empty(pages, 64, heads, dim, dim, device=DEV)
    assert cache.keys.numel() * 2 > 1 << 31 and cache.keys.nbytes + cache.values.nbytes > 5 * (1 << 30) - 1
    _, k, v = (t.contiguous() for t in _inputs(4, 8, heads, dim, dim, torch.bfloat16))
    slots = torch.tensor([pages * 64 - 1, 0, pages * 64 - 100, pages * 64], device=DEV)
    append_tokens(cache, k, v, slots)
    got = cache.gather(slots[:3])
    assert torch.equal(got[0], k[:3]) and torch.equal(got[1], v[:3])


def test_refusals():
    q, k, v = (t.contiguous() for t in _inputs(4, 4, 2, 64, 64, torch.bfloat16))
    cache, slots = make_cache(2, 16, 2, 64, 64, torch.bfloat16, fill=0.0), torch.arange(4, device=DEV)
    freq = rotary_frequencies(64, device=DEV)[0]
    for args, kw, text in (((k[:, :1], v, slots), {}, "k of shape"), ((k, v[:3], slots), {}, "v of shape"), ((k.half(), v.half(), slots), {}, "a cache of"), ((k, v.half(), slots), {}, "v is"),
                           ((k, v, slots[:3]), {}, "slots of shape"), ((k, v, slots.float()), {}, "not int64"), ((k, v, slots.cpu()), {}, "slots on"), ((k, v, slots), dict(positions=slots), "go together"),
                           ((k, v, slots), dict(q=q), "go together"), ((k, v, slots), dict(positions=slots, inv_freq=freq[:12]), "multiple of 8"),
                           ((k, v, slots), dict(positions=slots, inv_freq=freq, q=q[..., :32]), "q of shape"), ((k.clone().requires_grad_(True), v, slots), {}, "no_grad"),
                           ((k, v, slots), dict(positions=slots, inv_freq=torch.cat([freq, freq])), "inv_freq is"), ((k.float(), v.float(), slots), {}, "bfloat16 or float16")):
        with pytest.raises(ValueError, match=text):
            append_tokens(cache, *args, **kw)
    assert (cache.keys == 0).all() and (cache.values == 0).all()
    leaf = k.clone().requires_grad_(True)
    with torch.no_grad():
        append_tokens(cache, leaf, v, slots)
    assert torch.equal(cache.gather(slots)[0], k)


@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
def test_more_tokens_than_a_launch_has(kept8):
    tokens, dim = (1 << 22) + 1013, 32 if kept8 else 8
    g = torch.Generator(device=DEV).manual_seed(0)
    cache = PagedCache.empty((tokens + 1023) // 1024, 1024, 1, dim, kept8=kept8)
    slots = torch.randperm(tokens, generator=g, device=DEV)
    k, v = (torch.randint(-8, 9, (tokens, 1, dim), generator=g, device=DEV).bfloat16() for _ in range(2))       # (exact in 8 bits)
    append_tokens(cache, k, v, slots)
    for part in (slice(0, 70000), slice(tokens - 70000, None)):
        got = cache.gather(slots[part])
        assert torch.equal(got[0], k[part]) and torch.equal(got[1], v[part])
