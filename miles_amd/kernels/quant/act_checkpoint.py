"""Activations kept in 8 bits between the forward and the backward pass.

What a layer keeps for its backward pass is most of a training step's memory.  `checkpoint_activation` keeps it as MXFP8
(e4m3 codes, one E8M0 exponent byte for each 32 elements of a row, the layout of `mxfp8_quantize`): 1.03 bytes an element for
two or four.  `miles_amd.kernels.norm` and `miles_amd.kernels.linear` make such copies themselves (`checkpoint=True`), take one
that exists already, and read the codes in their backward passes without restoring the tensor in memory.

The scales are powers of two, so a restored bf16 or fp32 value is the code's value exactly; against the activation it is off
by at most half an e4m3 step, 2^-4 of the value (or 2^-10 of the group's scale, for the smallest).
"""

from __future__ import annotations

import math

import torch

from miles_amd import _lib, launch
from miles_amd._host import native
from miles_amd.utils.mxfp8 import MXFP8_GROUP_SIZE, mxfp8_dequantize


class ActCheckpoint:
    """An activation in 8 bits: `codes` float8_e4m3fn [..., K], `scales` uint8 [..., K/32], and the `dtype` it came in."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> None:
        self.codes, self.scales, self.dtype = codes, scales, dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    def restore(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values the codes stand for, in `dtype` (as they came, by default)."""
        return mxfp8_dequantize(self.codes, self.scales, self.dtype if dtype is None else dtype)

    def matrices(self, shape: torch.Size, device: torch.device, what: str) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes [M, K], scales [M, K/32]) for a kernel that takes them as the copy of a tensor of this shape on this device."""
        codes, scales = self.codes, self.scales
        if codes.shape != shape or codes.device != device or scales.device != device:
            raise ValueError(f"{what}: a checkpoint of shape {tuple(codes.shape)} on {codes.device} (scales on {scales.device}) for an input "
                             f"of shape {tuple(shape)} on {device}")
        check_width(shape[-1], what)
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.uint8 or scales.shape != (*shape[:-1], shape[-1] // MXFP8_GROUP_SIZE):
            raise ValueError(f"{what}: a checkpoint of {codes.dtype} codes and {scales.dtype} scales of shape {tuple(scales.shape)}, not of "
                             f"float8_e4m3fn codes and a uint8 scale for each {MXFP8_GROUP_SIZE} of a row")
        m = math.prod(shape[:-1])
        codes = codes.reshape(m, shape[-1]).contiguous()
        return codes if codes.data_ptr() % 16 == 0 else codes.clone(), scales.reshape(m, shape[-1] // MXFP8_GROUP_SIZE).contiguous()

    def __repr__(self) -> str:
        return f"ActCheckpoint(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.codes.device})"


def check_width(n: int, what: str) -> None:
    if n % MXFP8_GROUP_SIZE != 0:
        raise ValueError(f"{what}: {n} columns; activations are kept in 8 bits by groups of {MXFP8_GROUP_SIZE}")


def keep8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes and scales of x, made at once: also inside a `launch.deferred()` block, whose jobs run at its end."""
    k = x.shape[-1]
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((*x.shape[:-1], k // MXFP8_GROUP_SIZE), dtype=torch.uint8, device=x.device)
    launch.note_direct_call()
    with _lib.on_device(x.device):
        _lib.check(_lib.load().mq_mxfp8_quant(x.data_ptr(), _lib.dtype_code(x, "checkpoint_activation"), codes.data_ptr(), scales.data_ptr(),
                                              x.numel() // k if k else 0, k, _lib.stream_ptr(x.device)))
    return codes, scales


def checkpoint_activation(x: torch.Tensor) -> ActCheckpoint:
    """x [..., K] (bf16, fp16 or fp32, K a multiple of 32) kept in 8 bits.  The copy carries no gradient."""
    made = native.keep8(x)
    if made is not None:
        return ActCheckpoint(*made, x.dtype)
    _lib.require_gpu(x, "checkpoint_activation")
    _lib.dtype_code(x, "checkpoint_activation")
    if x.dim() == 0:
        raise ValueError("checkpoint_activation: expected a tensor with at least one dimension")
    check_width(x.shape[-1], "checkpoint_activation")
    return ActCheckpoint(*keep8(x.detach().contiguous()), x.dtype)
