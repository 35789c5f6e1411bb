"""A paged cache of keys and values, in 16 bits or in 8 (MXFP8 along each vector).

Pages have a fixed number of places; slot s is place s % page_size of page s // page_size, and which pages belong to which sequence is the
program's business (a table of page numbers, as `miles_amd.kernels.paged_attention` takes it).  `append_tokens` writes tokens into their
slots, keys rotated and both quantized on the way.

Layout: `values` [pages, heads, page_size, value_dim]; `keys` [pages, heads, key_dim / x, page_size, x], x the elements of 16 bytes: the
pieces of neighbouring tokens lie side by side, which is how the matrix instructions take them.  In 8 bits both are e4m3 codes with an
exponent byte for 32 elements, `key_scales` [pages, heads, key_dim / 32, page_size] and `value_scales` likewise.
"""

from __future__ import annotations

import ctypes

import torch

from miles_amd import _lib, launch
from miles_amd._host import native
from miles_amd.kernels._rows import wants_graph
from miles_amd.kernels.quant.act_checkpoint import MXFP8_GROUP_SIZE
from miles_amd.kernels.rotary import check_frequencies, check_positions
from miles_amd.utils.mxfp8 import mxfp8_dequantize

_HALVES = (torch.bfloat16, torch.float16)


class PagedCache:
    """The pages of one layer: `keys`, `values` and, in 8 bits, `key_scales`, `value_scales`, tensors of the module's layout."""

    __slots__ = ("keys", "values", "key_scales", "value_scales")

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor | None = None, value_scales: torch.Tensor | None = None) -> None:
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, key_dim: int, value_dim: int | None = None, *, dtype: torch.dtype = torch.bfloat16,
              kept8: bool = False, device="cuda") -> PagedCache:
        """Pages whose contents are whatever the memory held.  `kept8`: in 8 bits, for tensors of `dtype`."""
        value_dim = key_dim if value_dim is None else value_dim
        if dtype not in _HALVES:
            raise ValueError(f"PagedCache: bfloat16 or float16, got {dtype}")
        x = 16 if kept8 else 8
        if key_dim % x:
            raise ValueError(f"PagedCache: keys of {key_dim} elements, not a multiple of {MXFP8_GROUP_SIZE if kept8 else 8}")
        stored = torch.float8_e4m3fn if kept8 else dtype
        cache = cls(torch.empty((pages, kv_heads, key_dim // x, page_size, x), dtype=stored, device=device),
                    torch.empty((pages, kv_heads, page_size, value_dim), dtype=stored, device=device))
        if kept8:
            cache.key_scales, cache.value_scales = (torch.empty((pages, kv_heads, n // MXFP8_GROUP_SIZE, page_size), dtype=torch.uint8, device=device)
                                                    for n in (key_dim, value_dim))
        cache.check("PagedCache", dtype)
        return cache

    kept8 = property(lambda self: self.key_scales is not None)
    pages = property(lambda self: self.values.shape[0])
    kv_heads = property(lambda self: self.values.shape[1])
    page_size = property(lambda self: self.values.shape[2])
    value_dim = property(lambda self: self.values.shape[3])
    key_dim = property(lambda self: self.keys.shape[2] * self.keys.shape[4])

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in (self.keys, self.values, self.key_scales, self.value_scales) if t is not None)

    def check(self, what: str, dtype: torch.dtype) -> None:
        """Raises unless the tensors are a cache for tensors of `dtype`."""
        keys, values = self.keys, self.values
        if dtype not in _HALVES:
            raise ValueError(f"{what}: bfloat16 or float16 tensors, got {dtype}")
        if (self.key_scales is None) != (self.value_scales is None):
            raise ValueError(f"{what}: a cache with scales for both keys and values, or for neither")
        x, stored = (16, torch.float8_e4m3fn) if self.kept8 else (8, dtype)
        if values.dim() != 4 or keys.dim() != 5 or keys.shape[4] != x or (*keys.shape[:2], keys.shape[3]) != tuple(values.shape[:3]):
            raise ValueError(f"{what}: keys of shape {tuple(keys.shape)} and values of shape {tuple(values.shape)}; expected [pages, heads, key_dim/{x}, "
                             f"page_size, {x}] and [pages, heads, page_size, value_dim]")
        if keys.dtype != stored or values.dtype != stored:
            raise ValueError(f"{what}: a cache of {keys.dtype} keys and {values.dtype} values, expected {stored} for {dtype} tensors"
                             f"{' and 8-bit scales' if self.kept8 else ''}")
        for name, n in (("key_scales", self.key_dim), ("value_scales", self.value_dim)):
            scales = getattr(self, name)
            if scales is None:
                continue
            shape = (*values.shape[:2], n // MXFP8_GROUP_SIZE, values.shape[2])
            if n % MXFP8_GROUP_SIZE or tuple(scales.shape) != shape or scales.dtype != torch.uint8:
                raise ValueError(f"{what}: {name} are {scales.dtype} {tuple(scales.shape)} for vectors of {n} elements, expected uint8 {shape} and a multiple of "
                                 f"{MXFP8_GROUP_SIZE}")
        for t in (keys, values, self.key_scales, self.value_scales):
            if t is not None and (t.device != values.device or not t.is_contiguous() or t.requires_grad):
                raise ValueError(f"{what}: the tensors of a cache are contiguous, on one device and without gradients")
        if not self.page_size & (self.page_size - 1) == 0 or not 16 <= self.page_size <= 1024:
            raise ValueError(f"{what}: pages of {self.page_size} places; a power of two from 16 to 1024")
        for n in (self.key_dim, self.value_dim):
            if n % 8 or not 8 <= n <= 256:
                raise ValueError(f"{what}: vectors of {n} elements; a multiple of 8 up to 256")

    def struct(self, dtype: torch.dtype) -> _lib.Cache:
        address = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        return _lib.Cache(address(self.keys), address(self.values), address(self.key_scales), address(self.value_scales), self.pages, self.page_size,
                          self.kv_heads, self.key_dim, self.value_dim, _lib.DTYPE_CODE[dtype])

    def gather(self, slots: torch.Tensor, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(keys [..., heads, key_dim], values [..., heads, value_dim]) that lie in these slots, restored to `dtype` from 8 bits (bf16 by default).
        Slots outside of the cache raise; to see them, this waits for the device."""
        if slots.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"PagedCache.gather: slots are {slots.dtype}, not int64 or int32")
        if bool(((slots < 0) | (slots >= self.pages * self.page_size)).any()):
            raise IndexError(f"PagedCache.gather: a slot outside of the cache's {self.pages * self.page_size}")
        page, place = torch.div(slots, self.page_size, rounding_mode="floor"), slots % self.page_size
        n, flat = slots.shape, lambda t: t.reshape(-1)  # noqa: E731
        page, place = flat(page).long(), flat(place).long()
        raw = (lambda t: t.view(torch.uint8)) if self.kept8 else (lambda t: t)
        out = []
        for stored, scales in ((self.keys, self.key_scales), (self.values.unsqueeze(2), self.value_scales)):
            t = raw(stored)[page, :, :, place].flatten(2)
            if self.kept8:
                t = mxfp8_dequantize(t.contiguous().view(torch.float8_e4m3fn), scales[page, :, :, place].contiguous(), dtype or torch.bfloat16)
            out.append(t.reshape(*n, *t.shape[1:]))
        return out[0], out[1]

    def __repr__(self) -> str:
        return (f"PagedCache(pages={self.pages}, page_size={self.page_size}, kv_heads={self.kv_heads}, key_dim={self.key_dim}, value_dim={self.value_dim}, "
                f"dtype={self.keys.dtype}, device={self.keys.device})")


def _vectors(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, dim] with every vector one run of memory that begins at a multiple of 16 bytes (a view where there is one)."""
    ok = (t.shape[2] <= 1 or t.stride(2) == 1) and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or t.stride(0) % 8 == 0) and (t.shape[1] <= 1 or t.stride(1) % 8 == 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def refuse_graph(what: str, *tensors: torch.Tensor | None) -> None:
    if wants_graph(*tensors):
        raise ValueError(f"{what}: no gradient goes through a cache; call it under torch.no_grad()")


def append_tokens(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, positions: torch.Tensor | None = None,
                  inv_freq: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0, q: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes the keys and values of tokens into their slots of `cache`.

    k [tokens, heads, key_dim] and v [tokens, heads, value_dim], bf16 or fp16; slots [tokens] int64 or int32.  A token whose slot is not one of the
    cache's (-1, say, for padding) is left out.  Slots differ from each other: of one that is given twice the contents are any mix of
    the two tokens.  With `inv_freq` the keys are turned by their `positions` as `miles_amd.kernels.rotary.rotary` does it (a multiple of 8 pairs),
    and so are the queries `q` [tokens, query heads, key_dim], which are returned (those of tokens that are left out among them); None without
    `q`.  Into an 8-bit cache go the fp32 results of the turn, rounded once.  Carries no gradient."""
    what = "append_tokens"
    if not torch.compiler.is_dynamo_compiling():
        made = native.append(cache.keys, cache.values, cache.key_scales, cache.value_scales, k, v, slots, positions, inv_freq, interleaved, scale, q)
        if made is not None:
            return None if made is True else made
    _lib.require_gpu(k, what)
    cache.check(what, k.dtype)
    if k.dim() != 3 or tuple(k.shape[1:]) != (cache.kv_heads, cache.key_dim):
        raise ValueError(f"{what}: k of shape {tuple(k.shape)} for a cache of {cache.kv_heads} heads of {cache.key_dim}")
    tokens = k.shape[0]
    shapes = {"v": (v, (tokens, cache.kv_heads, cache.value_dim)), "q": (q, (tokens, q.shape[1] if q is not None and q.dim() == 3 else -1, cache.key_dim))}
    for name, (t, shape) in shapes.items():
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise ValueError(f"{what}: {name} of shape {tuple(t.shape)} beside k of shape {tuple(k.shape)} and a cache of {cache.kv_heads} heads of "
                             f"{cache.key_dim} and {cache.value_dim}")
        if t.dtype != k.dtype or t.device != k.device:
            raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, k {k.dtype} on {k.device}")
    if cache.keys.device != k.device:
        raise ValueError(f"{what}: a cache on {cache.keys.device}, tokens on {k.device}")
    check_positions(slots, (tokens,), k.device, what, "slots")
    pairs = 0
    if (positions is None) != (inv_freq is None) or (q is not None and inv_freq is None):
        raise ValueError(f"{what}: positions and inv_freq go together, and queries are given to be turned")
    if inv_freq is not None:
        check_positions(positions, (tokens,), k.device, what)
        check_frequencies(inv_freq, k.device, cache.key_dim, what)
        pairs = inv_freq.shape[0]
        if pairs % 8:
            raise ValueError(f"{what}: {pairs} pairs; a multiple of 8 (`rotary` turns any number)")
        positions, inv_freq = positions.expand(tokens).contiguous(), inv_freq.contiguous()
    refuse_graph(what, k, v, q)
    slots = slots.expand(tokens).contiguous()
    k, v = _vectors(k), _vectors(v)
    turned = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    q = None if q is None else _vectors(q)
    heads = lambda t, out=None: _lib.Heads(t.data_ptr(), out, t.shape[1], 0, t.stride(0), t.stride(1))  # noqa: E731
    args = [cache.struct(k.dtype), heads(k), heads(v), None if q is None else heads(q, turned.data_ptr())]
    is64 = lambda t, wide: int(t is not None and t.dtype == wide)  # noqa: E731
    address = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    launch.note_direct_call()
    for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales):
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)         # written in place: a graph that saved it before says so
    with _lib.on_device(k.device):
        _lib.check(_lib.load().mq_cache_append(
            *(None if a is None else ctypes.addressof(a) for a in args), tokens, slots.data_ptr(), is64(slots, torch.int64), address(positions),
            is64(positions, torch.int64), address(inv_freq), is64(inv_freq, torch.float64), pairs, int(bool(interleaved)), float(scale), _lib.stream_ptr(k.device)))
    return turned
