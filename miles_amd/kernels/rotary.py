"""Rotary positions with their backward pass.

Pairs of a vector's elements are turned by the angle position x inv_freq.  Angles, cosines and sines are computed in 64 bits for every token,
so that there is no table and no last position, and the heads of a token share them.  The backward pass turns by the negative angle; it is as
linear as the forward pass, and gradients of gradients are what they are.  `miles_amd.kernels.paged_cache.append_tokens` does the
same to keys and queries on their way into a cache.
"""

from __future__ import annotations

import ctypes
import math

import torch

from miles_amd import _lib, launch
from miles_amd._host import native
from miles_amd.kernels._rows import unpacked, wants_graph

# names that a kind of scaling needs and those that it may have; names that repeat what is known or change nothing
_SCALINGS = {"default": (set(), {"factor"}), "linear": ({"factor"}, set()),
             "yarn": ({"factor", "original_max_position_embeddings"}, {"beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"})}
_ANY_SCALING = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings", "max_position_embeddings"}


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: dict | None = None, device="cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq [dim/2] fp64, scale): the radians that each pair of `dim` elements turns by from one position to the next, `base`^(-2i/dim),
    and what cosines and sines are multiplied with, for `rotary(..., inv_freq, scale=scale)`.

    `scaling` stretches a context, with the names of a checkpoint's configuration (`rope_type` or `type`): {"rope_type": "linear", "factor"} divides every
    frequency by the factor; {"rope_type": "yarn", "factor", "original_max_position_embeddings"} keeps pairs that turn more than `beta_fast` (32) times in
    the original context, divides those that turn less than `beta_slow` (1) times, with a ramp between, whose ends are whole pairs unless `truncate` is
    False (Peng et al., "YaRN: Efficient context window extension of large language models", 2023).  YaRN's scale is `attention_factor`; without it
    m(`mscale`) / m(`mscale_all_dim`) where both are given, else m(1), with m(x) = 0.1 x ln(factor) + 1.  (Where a model multiplies its attention's scale
    by m(mscale_all_dim)^2 as well, that is the attention's argument.)  `rope_theta` has to be the base that is given, and `partial_rotary_factor` 1:
    `dim` is what turns.  Other names are refused, since they would change the result."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: an even number of elements, got {dim}")
    inv_freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    given = {} if scaling is None else {k: v for k, v in scaling.items() if v is not None}
    kind = given.get("rope_type", given.get("type", "default"))
    if kind not in _SCALINGS:
        raise ValueError(f"rotary_frequencies: unknown rope_type {kind!r}: linear or yarn (or an inv_freq of one's own)")
    needed, optional = _SCALINGS[kind]
    unknown = given.keys() - _ANY_SCALING - needed - optional
    if unknown or not needed <= given.keys():
        raise ValueError(f"rotary_frequencies: rope_type {kind!r} with {', '.join(sorted(map(str, unknown)))}, which is not known" if unknown else
                         f"rotary_frequencies: rope_type {kind!r} without {', '.join(sorted(needed - given.keys()))}")
    if given.get("rope_theta", base) != base or given.get("partial_rotary_factor", 1) != 1:
        raise ValueError(f"rotary_frequencies: a base of {base} and {dim} elements that turn, beside a rope_theta of {given.get('rope_theta')} and a partial_rotary_factor "
                         f"of {given.get('partial_rotary_factor')}; give them as base and dim")
    if kind == "default":
        return inv_freq.to(device), 1.0
    factor = float(given["factor"])
    if kind == "linear":
        return (inv_freq / factor).to(device), 1.0
    length, truncate = given["original_max_position_embeddings"], given.get("truncate", True)
    if not isinstance(truncate, bool):
        raise ValueError(f"rotary_frequencies: truncate is {truncate!r}, neither True nor False")

    def pair_that_turns(times: float) -> float:
        return dim * math.log(length / (times * 2 * math.pi)) / (2 * math.log(base))

    low, high = pair_that_turns(given.get("beta_fast") or 32), pair_that_turns(given.get("beta_slow") or 1)
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    slowed = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return (inv_freq * (1 - slowed) + inv_freq / factor * slowed).to(device), _yarn_scale(factor, given)


def _yarn_scale(factor: float, given: dict) -> float:
    if "attention_factor" in given:
        return float(given["attention_factor"])

    def m(x: float) -> float:
        return 0.1 * x * math.log(factor) + 1.0 if factor > 1 else 1.0

    over, under = given.get("mscale", 1.0), given.get("mscale_all_dim", 0.0)
    if "mscale" in given and over and under:
        return m(over) / m(under)
    if over == 1 and not under or factor <= 1:
        return m(1.0)
    raise ValueError(f"rotary_frequencies: mscale {given.get('mscale')} with mscale_all_dim {given.get('mscale_all_dim')}: one of the two alone has no meaning that programs "
                     "agree on; give both or an attention_factor")


def check_frequencies(inv_freq: torch.Tensor, device: torch.device, dim: int, what: str) -> None:
    if inv_freq.dtype not in (torch.float64, torch.float32) or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > dim:
        raise ValueError(f"{what}: inv_freq is {inv_freq.dtype} {tuple(inv_freq.shape)}; float64 or float32, one for each of at most {dim // 2} pairs")
    if inv_freq.device != device:
        raise ValueError(f"{what}: inv_freq on {inv_freq.device}, the input on {device}")
    if inv_freq.requires_grad:
        raise ValueError(f"{what}: inv_freq has no gradient")


def check_positions(positions: torch.Tensor, shape, device: torch.device, what: str, name: str = "positions") -> None:
    if positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: {name} are {positions.dtype}, not int64 or int32")
    if positions.device != device:
        raise ValueError(f"{what}: {name} on {positions.device}, the input on {device}")
    try:
        fits = torch.broadcast_shapes(positions.shape, shape) == torch.Size(shape)
    except RuntimeError:
        fits = False
    if not fits:
        raise ValueError(f"{what}: {name} of shape {tuple(positions.shape)} for tokens of shape {tuple(shape)}")


def _tokens(x: torch.Tensor) -> torch.Tensor:
    """x [..., heads, dim] as [batch, tokens, heads, dim] with the elements of a vector one behind the other (a view where there is one)."""
    if x.dim() != 4:
        x = x.unsqueeze(0) if x.dim() == 3 else x.reshape(1, math.prod(x.shape[:-2]), *x.shape[-2:])
    return x if x.shape[3] <= 1 or x.stride(3) == 1 else x.contiguous()


def _turn(tensors, positions, inv_freq, interleaved, scale, back):
    """The turned tensors, contiguous; None for None."""
    given = [t for t in tensors if t is not None]
    first = given[0]
    lead = first.shape[:-2]
    views = [_tokens(t) for t in given]
    batch, tokens = views[0].shape[:2]
    positions = positions.expand(lead)
    if first.dim() != 4 or (tokens > 1 and positions.stride(1) != 1):
        positions = positions.reshape(batch, tokens).contiguous()
    inv_freq = inv_freq.contiguous()
    outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in given]
    x = (_lib.Heads * len(given))(*(_lib.Heads(v.data_ptr(), o.data_ptr(), v.shape[2], v.stride(0), v.stride(1), v.stride(2)) for v, o in zip(views, outs)))
    launch.note_direct_call()
    with _lib.on_device(first.device):
        _lib.check(_lib.load().mq_rotary(
            ctypes.addressof(x), len(given), _lib.DTYPE_CODE[first.dtype], batch, tokens, first.shape[-1], positions.data_ptr(),
            int(positions.dtype == torch.int64), positions.stride(0), inv_freq.data_ptr(), int(inv_freq.dtype == torch.float64), inv_freq.shape[0],
            int(interleaved), scale, int(back), _lib.stream_ptr(first.device)))
    outs = iter(outs)
    return tuple(None if t is None else next(outs) for t in tensors)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, scale, back):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq)
        ctx.saved = (positions.shape, positions.dtype, inv_freq.shape, inv_freq.dtype)
        ctx.how = interleaved, scale, back
        return _turn((q, k), positions, inv_freq, interleaved, scale, back)

    @staticmethod
    def backward(ctx, dq, dk):
        grads = [g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad)]
        some = next((g for g in grads if g is not None), None)
        if some is not None:
            shape, kind, pairs, freq = ctx.saved
            positions, inv_freq = (unpacked(t, s, d, some.device, "rotary") for t, s, d in zip(ctx.saved_tensors, (shape, pairs), (kind, freq)))
            interleaved, scale, back = ctx.how
            grads = _apply(*grads, positions, inv_freq, interleaved, scale, not back)
        return (*grads, None, None, None, None, None)


def _apply(q, k, positions, inv_freq, interleaved, scale, back):
    if wants_graph(q, k):
        return _Rotary.apply(q, k, positions, inv_freq, interleaved, scale, back)
    return _turn((q, k), positions, inv_freq, interleaved, scale, back)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           scale: float = 1.0, inverse: bool = False):
    """(q, k) with the first 2 len(inv_freq) elements of every vector turned: elements i and i + len(inv_freq), or (`interleaved`) 2i and
    2i + 1, by the angle position x inv_freq[i], and multiplied by `scale`.  The elements behind them stay as they are.

    q [..., heads, dim], k [..., key heads, dim] or None (the result is then q's alone), bf16, fp16 or fp32 of any strides, views of a fused
    projection's output among them; positions int64 or int32, of q's leading shape or one that is broadcast to it; inv_freq fp64 or fp32
    (`rotary_frequencies`).  `inverse` turns back by the same angles.  Products and sums are fp32, each rounded once."""
    what = "rotary"
    if not torch.compiler.is_dynamo_compiling():
        made = native.rotary(q, k, positions, inv_freq, interleaved, scale, inverse)      # ordinary tensors: graph node in native code
        if made is not None:
            return made
    _lib.require_gpu(q, what)
    _lib.dtype_code(q, what)
    if q.dim() < 2:
        raise ValueError(f"{what}: expected a tensor [..., heads, dim], got {tuple(q.shape)}")
    lead, dim = q.shape[:-2], q.shape[-1]
    if k is not None:
        if k.dim() != q.dim() or k.shape[:-2] != lead or k.shape[-1] != dim:
            raise ValueError(f"{what}: k of shape {tuple(k.shape)} beside q of shape {tuple(q.shape)}")
        if k.dtype != q.dtype or k.device != q.device:
            raise ValueError(f"{what}: k is {k.dtype} on {k.device}, q {q.dtype} on {q.device}")
    check_positions(positions, lead, q.device, what)
    check_frequencies(inv_freq, q.device, dim, what)
    q, k = _apply(q, k, positions, inv_freq, bool(interleaved), float(scale), bool(inverse))
    return q if k is None else (q, k)
