"""What rotary positions, the paged cache and the attention over it refuse, and where they read of a cache (no GPU needed)."""

import ctypes

import pytest
import torch

from miles_amd import _lib, _probes
from miles_amd.kernels.paged_attention import paged_attention
from miles_amd.kernels.paged_cache import PagedCache, append_tokens
from miles_amd.kernels.rotary import rotary, rotary_frequencies

BF16 = torch.bfloat16
P = 0x1000      # a pointer that no refused call follows


def _refused(rc, text):
    assert rc == -1 and text.encode() in _lib.load().mq_last_error(), (rc, _lib.load().mq_last_error())


def _cache(pages=4, page_size=16, heads=2, key_dim=64, value_dim=64, scales=None, dtype=0, keys=P, values=P, value_scales=...):
    return _lib.Cache(keys, values, scales, scales if value_scales is ... else value_scales, pages, page_size, heads, key_dim, value_dim, dtype)


def test_cpu_tensors_are_refused():
    q, positions, freq = torch.zeros(4, 2, 64, dtype=BF16), torch.arange(4), rotary_frequencies(64, device="cpu")[0]
    cache = PagedCache.empty(2, 16, 2, 64, device="cpu")
    for call in (lambda: rotary(q, None, positions, freq), lambda: append_tokens(cache, q, q, positions),
                 lambda: paged_attention(q, cache, torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32))):
        with pytest.raises(_lib.MilesQuantError, match="GPU"):
            call()


@pytest.mark.parametrize("kw,text", [(dict(page_size=24), "power of two"), (dict(page_size=8), "power of two"), (dict(key_dim=320), "multiple of 8"),
                                     (dict(key_dim=60), "multiple of 8"), (dict(key_dim=48, kept8=True), "multiple of 32"), (dict(dtype=torch.float32), "bfloat16")])
def test_caches_that_are_none(kw, text):
    with pytest.raises(ValueError, match=text):
        PagedCache.empty(**{**dict(pages=2, page_size=16, kv_heads=2, key_dim=64, device="cpu"), **kw})


def test_tensors_that_are_no_cache():
    made = PagedCache.empty(3, 16, 2, 64, 96, kept8=True, device="cpu")
    made.check("a cache", BF16)
    assert (made.pages, made.page_size, made.kv_heads, made.key_dim, made.value_dim, made.kept8) == (3, 16, 2, 64, 96, True)
    assert made.nbytes == 3 * 16 * 2 * (64 + 96) * 33 // 32
    k, v, ks, vs = made.keys, made.values, made.key_scales, made.value_scales
    for tensors, text in (((k, v), "float16|bfloat16|expected"), ((k, v, ks), "for neither"), ((k, v[..., :64], ks, vs), "value_scales"), ((k, v, ks[:2], vs), "key_scales"),
                          ((k, v, ks.int(), vs), "uint8"), ((k[:2], v, ks, vs), "keys of shape"), ((k.half(), v, ks, vs), "a cache of"),
                          ((k.transpose(0, 1).contiguous().transpose(0, 1), v, ks, vs), "contiguous"), ((k, v.to("meta"), ks, vs), "one device")):
        with pytest.raises(ValueError, match=text):
            PagedCache(*tensors).check("a cache", BF16)


def test_gathered_slots():
    cache = PagedCache.empty(3, 16, 2, 8, device="cpu")
    cache.keys.copy_(torch.arange(48).view(3, 1, 1, 16, 1).expand_as(cache.keys))
    cache.values.copy_(torch.arange(48).view(3, 1, 16, 1).expand_as(cache.values))
    slots = torch.tensor([[0, 47], [16, 31]], dtype=torch.int32)
    k, v = cache.gather(slots)
    assert k.shape == v.shape == (2, 2, 2, 8) and torch.equal(k[..., 0, 0].int(), slots) and torch.equal(v[..., 1, 7].int(), slots)
    for bad in (-1, 48, 1 << 40):
        with pytest.raises(IndexError, match="outside"):
            cache.gather(torch.tensor([0, bad]))
    with pytest.raises(ValueError, match="int64 or int32"):
        cache.gather(torch.zeros(2))


def test_frequencies():
    f, scale = rotary_frequencies(128, 1e6, device="cpu")
    assert f.dtype == torch.float64 and scale == 1.0 and f[0] == 1.0 and abs(f[-1].item() - 1e6 ** (-126 / 128)) < 1e-18
    g, scale = rotary_frequencies(128, 1e6, scaling={"rope_type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(g, f / 4) and scale == 1.0
    yarn = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096}
    g, scale = rotary_frequencies(128, 1e6, scaling=yarn, device="cpu")
    turns = 4096 * f / (2 * torch.pi)
    assert torch.equal(g[turns > 33], f[turns > 33]) and torch.allclose(g[turns < 0.9], f[turns < 0.9] / 8, rtol=1e-15) and (g <= f).all() and (g >= f / 8).all()
    assert (g.diff() < 0).all() and abs(scale - (0.1 * torch.log(torch.tensor(8.0, dtype=torch.float64)).item() + 1)) < 1e-15
    assert rotary_frequencies(128, 1e6, scaling={**yarn, "attention_factor": 1.5}, device="cpu")[1] == 1.5
    with pytest.raises(ValueError, match="even number"):
        rotary_frequencies(7, device="cpu")
    with pytest.raises(ValueError, match="rope_type"):
        rotary_frequencies(8, scaling={"rope_type": "other", "factor": 2}, device="cpu")


def test_c_entry_of_rotary_positions():
    f = _lib.load().mq_rotary

    def call(n=1, dtype=0, batch=1, tokens=4, dim=64, positions=P, freq=P, pairs=32, inp=P, heads=2, x=True):
        x = (_lib.Heads * 2)(_lib.Heads(inp, P, heads, 0, 128, 64), _lib.Heads(inp, P, heads, 0, 128, 64)) if x else None
        return f(None if x is None else ctypes.addressof(x), n, dtype, batch, tokens, dim, positions, 1, 0, freq, 1, pairs, 0, 1.0, 0, None)

    _refused(call(x=False), "bad argument")
    _refused(call(n=3), "bad argument")
    _refused(call(dtype=3), "bad argument")
    _refused(call(pairs=33), "bad argument")
    _refused(call(tokens=-1), "bad argument")
    _refused(call(dim=2048, pairs=0), "1024")
    _refused(call(batch=1 << 20, tokens=1 << 20), "too large")
    _refused(call(heads=1 << 16), "too large")
    _refused(call(positions=None), "null pointer")
    _refused(call(inp=None), "null pointer")
    assert call(tokens=0) == 0 and call(heads=0) == 0


def test_c_entry_that_appends():
    f = _lib.load().mq_cache_append

    def call(cache=None, heads=2, v_heads=2, k=P, v=P, q=None, tokens=4, slots=P, positions=P, freq=P, pairs=32, stride=128):
        cache = cache or _cache()
        k, v = _lib.Heads(k, None, heads, 0, stride, 64), _lib.Heads(v, None, v_heads, 0, 128, 64)
        return f(ctypes.addressof(cache), ctypes.addressof(k), ctypes.addressof(v), None if q is None else ctypes.addressof(q), tokens, slots, 1, positions, 1, freq, 1, pairs, 0,
                 1.0, None)

    for cache, text in ((_cache(page_size=24), "power of two"), (_cache(page_size=8), "power of two"), (_cache(key_dim=264), "8 to 256"), (_cache(key_dim=60), "multiple of 8"),
                        (_cache(scales=P, value_dim=48), "multiple of 32"), (_cache(scales=P, value_scales=None), "for neither"), (_cache(dtype=2), "bf16 or fp16"),
                        (_cache(keys=None), "null pointer"), (_cache(values=P + 8), "16 bytes"), (_cache(heads=60000, page_size=1024), "too large"), (_cache(pages=-1), "bad argument")):
        _refused(call(cache), text)
    _refused(call(heads=3), "as many heads")
    _refused(call(v_heads=1), "as many heads")
    _refused(call(pairs=12), "multiple of 8")
    _refused(call(pairs=40), "bad argument")
    _refused(call(slots=None), "null pointer")
    _refused(call(positions=None), "null pointer")
    _refused(call(k=P + 2), "16 bytes")
    _refused(call(stride=132), "16 bytes")
    _refused(call(q=_lib.Heads(P, P + 4, 8, 0, 512, 64)), "16 bytes")
    _refused(call(q=_lib.Heads(P, None, 8, 0, 512, 64)), "null pointer")
    assert call(tokens=0) == 0


def test_c_entry_of_the_attention():
    lib = _lib.load()
    size = ctypes.c_int64(-1)

    def workspace(cache=None, batch=2, heads=4, width=4, window=0, out=ctypes.addressof(size)):
        cache = cache or _cache()
        return lib.mq_paged_attention_workspace(ctypes.addressof(cache), batch, heads, width, window, out)

    def call(cache=None, q=P, stride=256, table=P, lengths=P, out=P, batch=2, heads=4, width=4, window=0, ws=P):
        cache = cache or _cache()
        return lib.mq_paged_attention(ctypes.addressof(cache), q, stride, 64, table, width, width, lengths, None, 0.125, window, out, batch, heads, ws, None)

    for f in (workspace, call):
        _refused(f(heads=5), "the key heads divide")
        _refused(f(window=-1), "bad argument")
        _refused(f(batch=-1), "bad argument")
        _refused(f(width=1 << 31), "too large")
        _refused(f(batch=1 << 20, width=1 << 20), "too large")
        _refused(f(_cache(page_size=48)), "power of two")
    _refused(workspace(out=None), "null pointer")
    _refused(call(q=None), "null pointer")
    _refused(call(table=None), "null pointer")
    _refused(call(q=P + 2), "16 bytes")
    _refused(call(stride=260), "16 bytes")
    # no sequence can be long: no partial results; else they need their memory, at most as much as the card has workgroups for
    assert workspace() == 0 and size.value == 0
    assert workspace(width=1 << 16) == 0 and 0 < size.value < 64 << 20
    assert workspace(width=1 << 16, window=100) == 0 and size.value == 0
    _refused(call(width=1 << 16, ws=None), "null pointer")
    _refused(call(width=1 << 16, ws=P + 4), "16 bytes")
    assert call(batch=0) == 0 and call(heads=0) == 0


def _places(id, pages, length, capacity, window, tile, half, key_row, value_row, shift):
    out = (ctypes.c_int64 * 8)()
    assert _probes.load().mqp_paged_places(id, pages, length, capacity, window, tile, half, key_row, value_row, shift, ctypes.addressof(out)) == 0
    return list(out)


@pytest.mark.parametrize("shift", [4, 5, 8])
@pytest.mark.parametrize("length,window", [(0, 0), (-5, 0), (1, 0), (16, 0), (17, 3), (33, 0), (100, 40), (100, 1), (1000, 0), (2**31 - 1, 7), (300, 290)])
def test_nothing_outside_of_a_cache_is_read(length, window, shift):
    """Whatever numbers a table holds: what a step may read lies inside the page, and inside what is seen."""
    pages, capacity, key_row, value_row = 7, 512, 256, 128
    ids = [0, 3, 6, 7, 8, -1, -7, 2**31 - 1, -(2**31)]
    lo, hi, tiles = _places(0, pages, length, capacity, window, 0, 0, key_row, value_row, shift)[:3]
    assert hi == min(max(length, 0), capacity) and lo == min(max(length - window, 0) if window else 0, hi)
    seen = set()
    for tile in range(tiles + 2):
        for half in range(2):
            first = lo // 32 * 32 + tile * 32 + half * 16
            for id in ids:
                _, _, _, some, page, place, keys, values = _places(id, pages, length, capacity, window, tile, half, key_row, value_row, shift)
                inside = 0 <= id < pages and tile < tiles and first < hi and first + 16 > lo
                assert some == inside and page == (id if inside else 0) and place == first % (1 << shift)
                if not inside:
                    assert keys == values == 0
                    continue
                assert 0 < keys and place * 16 + keys == key_row << shift and place + 16 <= 1 << shift
                assert values == min(16, hi - first) * value_row and place * value_row + values <= value_row << shift
            if tile < tiles:
                seen |= set(range(max(first, lo), min(first + 16, hi)))
    assert seen == set(range(lo, hi))


def test_slots_outside_of_a_cache():
    f = _probes.load().mqp_paged_slot
    assert [f(s, 64) for s in (-(2**63), -1, 0, 63, 64, 2**40, 2**63 - 1)] == [0, 0, 1, 1, 0, 0, 0] and f(0, 0) == 0
