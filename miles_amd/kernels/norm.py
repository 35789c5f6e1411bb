"""Layer norm and RMS norm with their backward passes.

Rows of bf16, fp16 or fp32 of any length; statistics and sums are fp32.  For the backward pass a norm keeps its input and a
statistic or two for each row, or (`checkpoint=True`) the normalized values in 8 bits, from which the backward pass works
directly.  `output_checkpoint=True` also returns the 8-bit copy of the result that the next layer keeps as its input
(`miles_amd.kernels.linear.linear(..., checkpoint=copy)`), made in the same pass.

Gradients are deterministic: the rows' sums are added in an order that depends on the sizes alone.  They can be taken once
(there is no gradient of a gradient).
"""

from __future__ import annotations

import torch

from miles_amd import _lib, launch
from miles_amd._host import native
from miles_amd.kernels._rows import address, gradients_once, one_run, pitch, rows_like_contiguous, unpacked, wants_graph
from miles_amd.kernels.quant.act_checkpoint import MXFP8_GROUP_SIZE, ActCheckpoint, check_width


def _empty8(m: int, n: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty((m, n), dtype=torch.float8_e4m3fn, device=device),
            torch.empty((m, n // MXFP8_GROUP_SIZE), dtype=torch.uint8, device=device))


def _forward(x, weight, bias, eps, rms, statistics, keep, copy):
    """(y, mean, rstd, kept xhat, its scales, copy of y, its scales), with None for what is not asked for."""
    x2 = rows_like_contiguous(x)
    m, n = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = torch.empty(m, dtype=torch.float32, device=x.device) if statistics and not rms and not keep else None
    rstd = torch.empty(m, dtype=torch.float32, device=x.device) if statistics else None
    xq, xs = _empty8(m, n, x.device) if keep else (None, None)
    yq, ys = _empty8(m, n, x.device) if copy else (None, None)
    vector = weight if weight is not None else bias
    launch.note_direct_call()
    with _lib.on_device(x.device):
        _lib.check(_lib.load().mq_norm_forward(
            x2.data_ptr(), _lib.DTYPE_CODE[x.dtype], pitch(x2), address(weight), address(bias),
            _lib.DTYPE_CODE[x.dtype if vector is None else vector.dtype], y.data_ptr(), address(xq), address(xs), address(yq), address(ys),
            address(mean), address(rstd), m, n, eps, int(rms), _lib.stream_ptr(x.device)))
    return y, mean, rstd, xq, xs, yq, ys


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rms, keep, copy):
        y, mean, rstd, xq, xs, yq, ys = _forward(x, weight, bias, eps, rms, True, keep, copy)
        ctx.save_for_backward(xq if keep else x, xs, mean, rstd, weight)
        ctx.rms, ctx.shape = rms, x.shape
        ctx.vector = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        if copy:
            ctx.mark_non_differentiable(yq, ys)
        return y, yq, ys

    @staticmethod
    @gradients_once("norm")
    def backward(ctx, dy, *_):
        x, xs, mean, rstd, weight = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dy2 = rows_like_contiguous(dy)
        m, n = dy2.shape
        vector = ctx.vector
        saved = lambda t, shape, dtype: unpacked(t, shape, dtype, dy.device, "norm")  # noqa: E731
        if xs is not None:
            x2 = one_run(saved(x, (m, n), torch.float8_e4m3fn))
            xs = one_run(saved(xs, (m, n // MXFP8_GROUP_SIZE), torch.uint8))
        else:
            x2 = rows_like_contiguous(saved(x, ctx.shape, dy.dtype))
        mean, rstd, weight = (one_run(saved(t, shape, dtype)) for t, shape, dtype in
                              ((mean, (m,), torch.float32), (rstd, (m,), torch.float32), (weight, (n,), vector)))
        lib = _lib.load()
        launch.note_direct_call()
        dx = torch.empty(ctx.shape, dtype=dy.dtype, device=dy.device) if want_x else None
        dw = torch.empty(n, dtype=vector, device=dy.device) if want_w else None
        db = torch.empty(n, dtype=vector, device=dy.device) if want_b else None
        sums = int(want_w) + int(want_b)
        ws = torch.empty(sums * lib.mq_norm_backward_parts(m, n) * n, dtype=torch.float32, device=dy.device) if sums else None
        with _lib.on_device(dy.device):
            _lib.check(lib.mq_norm_backward(
                dy2.data_ptr(), _lib.DTYPE_CODE[dy.dtype], pitch(dy2), x2.data_ptr(), pitch(x2), address(xs), address(mean), rstd.data_ptr(),
                address(weight), _lib.DTYPE_CODE[vector], address(dx), address(dw), address(db), address(ws), m, n, int(ctx.rms),
                _lib.stream_ptr(dy.device)))
        return dx, dw, db, None, None, None, None


def _norm(what, x, weight, bias, eps, rms, checkpoint, output_checkpoint):
    if not torch.compiler.is_dynamo_compiling():
        made = native.norm(x, weight, bias, eps, rms, checkpoint, output_checkpoint)      # ordinary tensors: graph node in native code
        if made is not None:
            return (made[0], ActCheckpoint(made[1], made[2], x.dtype)) if output_checkpoint else made
    _lib.require_gpu(x, what)
    _lib.dtype_code(x, what)
    if x.dim() == 0:
        raise ValueError(f"{what}: expected a tensor with at least one dimension")
    n = x.shape[-1]
    for name, v in (("weight", weight), ("bias", bias)):
        if v is None:
            continue
        if v.shape != (n,):
            raise ValueError(f"{what}: {name} of shape {tuple(v.shape)} for rows of {n}")
        if v.device != x.device:
            raise ValueError(f"{what}: {name} on {v.device}, the input on {x.device}")
        if v.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: {name} is {v.dtype}; it has the input's type ({x.dtype}) or is float32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{what}: weight is {weight.dtype}, bias {bias.dtype}")
    if checkpoint or output_checkpoint:
        check_width(n, what)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    eps, rms, copy = float(eps), bool(rms), bool(output_checkpoint)
    if wants_graph(x, weight, bias):
        y, yq, ys = _Norm.apply(x, weight, bias, eps, rms, bool(checkpoint), copy)
    else:
        y, _mean, _rstd, _xq, _xs, yq, ys = _forward(x, weight, bias, eps, rms, False, False, copy)
    if not copy:
        return y
    return y, ActCheckpoint(yq.view(x.shape), ys.view(*x.shape[:-1], n // MXFP8_GROUP_SIZE), x.dtype)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5, *,
               checkpoint: bool = False, output_checkpoint: bool = False):
    """`(x - mean) / sqrt(var + eps) * weight + bias` over the last dimension.

    x [..., n] bf16, fp16 or fp32; weight and bias [n] of x's type or fp32, both of one type.  `checkpoint`: keep the
    normalized values in 8 bits for the backward pass instead of x (n a multiple of 32).  `output_checkpoint`: return
    `(y, ActCheckpoint of y)`."""
    return _norm("layer_norm", x, weight, bias, eps, False, checkpoint, output_checkpoint)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *, checkpoint: bool = False,
             output_checkpoint: bool = False):
    """`x / sqrt(mean(x^2) + eps) * weight` over the last dimension; arguments as those of `layer_norm`."""
    return _norm("rms_norm", x, weight, None, eps, True, checkpoint, output_checkpoint)
