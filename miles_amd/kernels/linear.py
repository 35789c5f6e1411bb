"""Linear layers with bias, activation and residual in the product's epilogue, and their backward passes.

The products run on the matrix cores with fp32 sums; one rounding makes the result.  In the backward pass of an activation, the
gradient of its argument is rounded to the tensors' type on its way into the two products behind it (in fp16 it is an infinity
beyond 65504), not in the bias's gradient.  For the backward pass a layer keeps its
input and, where it has an activation, what that is applied to: both as they are, or (`checkpoint=True`) both in 8 bits.  The
weight's gradient is then taken from the codes directly, whose values are exact in bf16.  Gradients are deterministic and can
be taken once (there is no gradient of a gradient).
"""

from __future__ import annotations

import ctypes
import math

import torch

from miles_amd import _lib, launch
from miles_amd._host import native
from miles_amd.kernels._rows import address, gradients_once, one_run, pitch, rows, unpacked, wants_graph
from miles_amd.kernels.quant.act_checkpoint import MXFP8_GROUP_SIZE, ActCheckpoint, check_width, keep8

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}      # MQ_ACT_*
_FORWARD, _INPUT_GRAD, _WEIGHT_GRAD = 0, 1, 2                                   # MQ_LINEAR_*


def _workspace(product: int, a: torch.Tensor, b: torch.Tensor, kept8: bool, m: int, n: int, k: int) -> torch.Tensor | None:
    """Scratch memory of a product of two matrices as they are passed to it, or None."""
    size = ctypes.c_int64()
    _lib.check(_lib.load().mq_linear_workspace(product, a.data_ptr(), pitch(a), b.data_ptr(), pitch(b), int(kept8), m, n, k, ctypes.addressof(size)))
    return torch.empty(size.value, dtype=torch.uint8, device=a.device) if size.value else None


def _forward(x2, weight, bias, act, residual2, keep_z, keep8_z):
    """(y [M, N], z or its codes, scales of the codes)"""
    (m, k), n = x2.shape, weight.shape[0]
    device = x2.device
    y = torch.empty((m, n), dtype=x2.dtype, device=device)
    z = scales = None
    if keep_z:
        z = torch.empty((m, n), dtype=torch.float8_e4m3fn if keep8_z else x2.dtype, device=device)
        scales = torch.empty((m, n // MXFP8_GROUP_SIZE), dtype=torch.uint8, device=device) if keep8_z else None
    launch.note_direct_call()
    ws = _workspace(_FORWARD, x2, weight, keep_z and keep8_z, m, n, k)
    with _lib.on_device(device):
        _lib.check(_lib.load().mq_linear_forward(
            x2.data_ptr(), _lib.DTYPE_CODE[x2.dtype], pitch(x2), weight.data_ptr(), pitch(weight), address(bias), act, address(residual2),
            pitch(residual2) if residual2 is not None else 0, y.data_ptr(), address(None if keep8_z else z), address(z if keep8_z else None),
            address(scales), m, n, k, address(ws), _lib.stream_ptr(device)))
    return y, z, scales


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, checkpoint, codes, scales):
        x2, w2 = rows(x), rows(weight)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        y, z, z_scales = _forward(x2, w2, bias, act, rows(residual) if residual is not None else None,
                                  act != 0 and (need_x or need_w or need_b), checkpoint)
        kept = x_scales = None
        if need_w:
            if checkpoint:
                kept, x_scales = (codes, scales) if codes is not None else keep8(x2.contiguous())
            else:
                kept = x
        ctx.save_for_backward(kept, x_scales, z, z_scales, weight if need_x else None)
        ctx.act, ctx.x_shape, ctx.n, ctx.dtype = act, x.shape, weight.shape[0], x.dtype
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @gradients_once("linear")
    def backward(ctx, dy):
        kept, x_scales, z, z_scales, weight = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        n, k, device, dtype = ctx.n, ctx.x_shape[-1], dy.device, _lib.DTYPE_CODE[ctx.dtype]
        lib = _lib.load()
        launch.note_direct_call()
        dz = dy2 = rows(dy)
        m = dy2.shape[0]
        saved = lambda t, shape, dtype: unpacked(t, shape, dtype, device, "linear")  # noqa: E731
        if x_scales is not None:
            kept, x_scales = one_run(saved(kept, (m, k), torch.float8_e4m3fn)), one_run(saved(x_scales, (m, k // MXFP8_GROUP_SIZE), torch.uint8))
        else:
            kept = saved(kept, ctx.x_shape, ctx.dtype)
        z = one_run(saved(z, (m, n), ctx.dtype if z_scales is None else torch.float8_e4m3fn))
        z_scales = one_run(saved(z_scales, (m, n // MXFP8_GROUP_SIZE), torch.uint8))
        weight = saved(weight, (n, k), ctx.dtype)
        with _lib.on_device(device):
            stream = _lib.stream_ptr(device)
            if need_b or (ctx.act and (need_x or need_w)):
                dz = torch.empty((m, n), dtype=ctx.dtype, device=device) if ctx.act else None
                db = torch.empty(n, dtype=ctx.dtype, device=device) if need_b else None
                ws = torch.empty(lib.mq_activation_backward_parts(m, n) * n, dtype=torch.float32, device=device) if need_b else None
                _lib.check(lib.mq_activation_backward(dy2.data_ptr(), dtype, pitch(dy2), address(z), address(z_scales), ctx.act, address(dz),
                                                      address(db), address(ws), m, n, stream))
                if dz is None:
                    dz = dy2
            if need_x:
                w2 = rows(weight)
                dx = torch.empty(ctx.x_shape, dtype=ctx.dtype, device=device)
                ws = _workspace(_INPUT_GRAD, dz, w2, False, m, n, k)
                _lib.check(lib.mq_linear_input_grad(dz.data_ptr(), dtype, pitch(dz), w2.data_ptr(), pitch(w2), dx.data_ptr(), m, n, k,
                                                    address(ws), stream))
            if need_w:
                x2 = kept if x_scales is not None else rows(kept)
                dw = torch.empty((n, k), dtype=ctx.dtype, device=device)
                ws = _workspace(_WEIGHT_GRAD, dz, x2, x_scales is not None, m, n, k)
                _lib.check(lib.mq_linear_weight_grad(dz.data_ptr(), dtype, pitch(dz), x2.data_ptr(), pitch(x2), address(x_scales),
                                                     dw.data_ptr(), m, n, k, address(ws), stream))
        return dx, dw, db, dy if need_r else None, None, None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None, checkpoint: bool | ActCheckpoint = False) -> torch.Tensor:
    """`activation(x @ weight.T + bias) + residual`, in one pass over the result.

    x [..., K], weight [N, K], bias [N], residual [..., N], all bf16 or all fp16; the result is [..., N].  `activation`: None,
    "relu", "silu", "gelu" or "gelu_tanh".  `checkpoint=True` keeps x (K a multiple of 32) and the activation's argument (N a
    multiple of 32) in 8 bits for the backward pass; an `ActCheckpoint` of x that exists already (of a norm's output, or one
    that several projections of one input share) is kept instead of a new one."""
    what = "linear"
    if activation in ACTIVATIONS and not torch.compiler.is_dynamo_compiling():
        given = type(checkpoint) is ActCheckpoint
        made = native.linear(x, weight, bias, ACTIVATIONS[activation], residual, given or checkpoint,          # ordinary tensors: graph
                             checkpoint.codes if given else None, checkpoint.scales if given else None)        # node in native code
        if made is not None:
            return made
    _lib.require_gpu(x, what)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"linear: bfloat16 or float16 tensors, got {x.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: unknown activation {activation!r}: one of {', '.join(map(repr, ACTIVATIONS))}")
    if x.dim() == 0 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"linear: weight of shape {tuple(weight.shape)} for an input of shape {tuple(x.shape)}")
    n, k = weight.shape
    shapes = {"weight": (weight, (n, k)), "bias": (bias, (n,)), "residual": (residual, (*x.shape[:-1], n))}
    for name, (t, shape) in shapes.items():
        if t is None:
            continue
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"linear: {name} of shape {tuple(t.shape)}, expected {tuple(shape)}")
        if t.dtype != x.dtype:
            raise ValueError(f"linear: {name} is {t.dtype}, the input {x.dtype}")
        if t.device != x.device:
            raise ValueError(f"linear: {name} on {t.device}, the input on {x.device}")
    act = ACTIVATIONS[activation]
    codes = scales = None
    if isinstance(checkpoint, ActCheckpoint):
        codes, scales = checkpoint.matrices(x.shape, x.device, what)
    elif checkpoint is not True and checkpoint is not False:
        raise ValueError(f"linear: checkpoint is True, False or an ActCheckpoint, got {type(checkpoint).__name__}")
    keep = checkpoint is not False
    if keep:
        check_width(k, what)
        if act:
            check_width(n, what)
    bias = bias.contiguous() if bias is not None else None
    if wants_graph(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act, keep, codes, scales)
    y = _forward(rows(x), rows(weight), bias, act, rows(residual) if residual is not None else None, False, False)[0]
    return y.view(*x.shape[:-1], n)
