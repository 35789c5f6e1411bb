"""Tensors as the row kernels take them: a matrix of rows, each with its elements one behind the other."""

from __future__ import annotations

import math

import torch


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
