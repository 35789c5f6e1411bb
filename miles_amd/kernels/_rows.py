"""Tensors as the row kernels take them: a matrix of rows, each with its elements one behind the other."""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from miles_amd._host import native


def wants_graph(*tensors: torch.Tensor | None) -> bool:
    """Whether a result of these tensors belongs to a graph; also where one carries a forward-mode derivative, which a graph node refuses."""
    given = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        return True
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in given)


def gradients_once(what: str):
    """For a `backward` whose gradients come out of kernels: where a graph of the backward pass itself is asked for
    (`create_graph=True`), they are part of one that refuses to be gone through.  They would pass for constants otherwise, also where
    the incoming gradient is one.  An incoming gradient that is handed on stays as it is."""
    def wrap(backward):
        @functools.wraps(backward)
        def once(ctx, *grads):
            again = torch.is_grad_enabled()
            with torch.no_grad():
                out = backward(ctx, *grads)
            if not again:
                return out
            given = [g for g in grads if g is not None]
            made = [o for o in out if o is not None and not any(o is g for g in given)]
            refused = dict(zip(map(id, made), native.once(made, given, what)))
            return tuple(refused.get(id(o), o) for o in out)
        return once
    return wrap


def unpacked(t: torch.Tensor | None, shape, dtype: torch.dtype, device: torch.device, what: str) -> torch.Tensor | None:
    """A tensor that was saved, as the kernels may read it: hooks on saved tensors may give back anything, and a kernel has no way to see it."""
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device):
        raise RuntimeError(f"{what}: a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}, not of the type, shape and device that "
                           f"it was saved with ({dtype} {tuple(shape)} on {device})")
    return t


def one_run(t: torch.Tensor | None) -> torch.Tensor | None:
    """t as one run of memory that begins at a multiple of 16 bytes."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def rows(t: torch.Tensor) -> torch.Tensor:
    """t [..., n] as a matrix whose rows may lie apart (a view where there is one; rows that overlap are copied)."""
    n = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), n)
    if (n > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < n):
        t = t.contiguous()
    return t


def pitch(t: torch.Tensor) -> int:
    """Elements from one row of a matrix to the next."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def rows_like_contiguous(t: torch.Tensor) -> torch.Tensor:
    """`rows(t)`, copied unless every row has the address modulo 16 bytes that it has in a contiguous tensor."""
    m = rows(t)
    if m.data_ptr() % 16 == 0 and (m.shape[0] <= 1 or (m.stride(0) - m.shape[1]) * m.element_size() % 16 == 0):
        return m
    return m.clone(memory_format=torch.contiguous_format)
