"""Attention of one new token for each of a batch of sequences over a paged cache.

Keys and values are read once, in 16 bits or from their 8-bit codes.  The work is shared out on the device by the sequences' lengths, so that one
long sequence among short ones keeps the whole card busy, and a call that was captured into a graph holds for other lengths and page tables.
Results of the same inputs are the same from run to run; where a sequence is cut depends on the lengths of the batch, and with it the order of its sums.
"""

from __future__ import annotations

import ctypes
import math

import torch

from miles_amd import _lib, launch
from miles_amd._host import native
from miles_amd.kernels.paged_cache import PagedCache, _vectors, refuse_graph


def paged_attention(q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                    window: int | None = None, sinks: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v over each sequence's tokens, [batch, heads, value_dim] of q's type.

    q [batch, heads, key_dim] bf16 or fp16, heads a multiple of the cache's (head h reads key head h // (heads / key heads)).  pages [batch, width] int32:
    the numbers of the pages that a sequence's tokens lie in, in their order; lengths [batch] int32: its tokens, the new one included.  Entries
    behind a sequence's last page are not read.  Tokens on a page that the cache has not, and tokens beyond the table's width, are left out;
    a sequence without a token (length 0: an idle place of the batch) gives zeros.  scale: 1 / sqrt(key_dim) by default.  window: the last
    `window` tokens alone are seen.  sinks [heads] fp32: a score that takes part in each head's softmax without a value.  Carries no gradient."""
    what = "paged_attention"
    if not torch.compiler.is_dynamo_compiling():
        made = native.attend(q, cache.keys, cache.values, cache.key_scales, cache.value_scales, pages, lengths, scale, window, sinks)
        if made is not None:
            return made
    _lib.require_gpu(q, what)
    cache.check(what, q.dtype)
    if q.dim() != 3 or q.shape[2] != cache.key_dim or q.shape[1] % cache.kv_heads:
        raise ValueError(f"{what}: q of shape {tuple(q.shape)} for a cache of {cache.kv_heads} heads of {cache.key_dim}")
    batch, heads = q.shape[:2]
    if pages.dim() != 2 or pages.shape[0] != batch or lengths.shape != (batch,):
        raise ValueError(f"{what}: pages of shape {tuple(pages.shape)} and lengths of shape {tuple(lengths.shape)} for {batch} sequences")
    if pages.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise ValueError(f"{what}: pages are {pages.dtype}, lengths {lengths.dtype}, both are int32")
    if sinks is not None and (sinks.shape != (heads,) or sinks.dtype != torch.float32):
        raise ValueError(f"{what}: sinks are {sinks.dtype} {tuple(sinks.shape)}, expected float32 {(heads,)}")
    if window is not None and window < 1:
        raise ValueError(f"{what}: a window of {window} tokens")
    for name, t in (("the cache", cache.keys), ("pages", pages), ("lengths", lengths), ("sinks", sinks)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{what}: {name} on {t.device}, q on {q.device}")
    refuse_graph(what, q, sinks)
    q = _vectors(q)
    if pages.shape[1] > 1 and pages.stride(1) != 1:
        pages = pages.contiguous()
    lengths = lengths.contiguous()
    sinks = None if sinks is None else sinks.contiguous()
    window = 0 if window is None else min(int(window), 1 << 62)
    scale = 1.0 / math.sqrt(cache.key_dim) if scale is None else float(scale)
    struct, size = cache.struct(q.dtype), ctypes.c_int64()
    out = torch.empty((batch, heads, cache.value_dim), dtype=q.dtype, device=q.device)
    launch.note_direct_call()
    lib = _lib.load()
    _lib.check(lib.mq_paged_attention_workspace(ctypes.addressof(struct), batch, heads, pages.shape[1], window, ctypes.addressof(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=q.device) if size.value else None
    with _lib.on_device(q.device):
        _lib.check(lib.mq_paged_attention(
            ctypes.addressof(struct), q.data_ptr(), q.stride(0), q.stride(1), pages.data_ptr(), pages.stride(0), pages.shape[1], lengths.data_ptr(),
            None if sinks is None else sinks.data_ptr(), scale, window, out.data_ptr(), batch, heads, None if ws is None else ws.data_ptr(),
            _lib.stream_ptr(q.device)))
    return out
