"""What the norms, linear layers and 8-bit activation checkpoints refuse, in Python and at the C entries (no GPU needed)."""

import ctypes

import pytest
import torch

from miles_amd import _lib
from miles_amd.kernels.linear import linear
from miles_amd.kernels.norm import layer_norm, rms_norm
from miles_amd.kernels.quant.act_checkpoint import ActCheckpoint, checkpoint_activation, check_width
from miles_amd.utils.mxfp8 import mxfp8_dequantize

BF16 = torch.bfloat16


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(32, 64, dtype=BF16)
    for call in (lambda: linear(x, w), lambda: layer_norm(x), lambda: rms_norm(x), lambda: checkpoint_activation(x),
                 lambda: mxfp8_dequantize(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8)),
                 lambda: ActCheckpoint(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8), BF16).restore()):
        with pytest.raises(_lib.MilesQuantError, match="GPU"):
            call()


def test_width_of_an_8_bit_copy():
    check_width(64, "linear")
    with pytest.raises(ValueError, match="groups of 32"):
        check_width(48, "linear")


def test_a_checkpoint_that_is_not_the_inputs():
    codes, scales = torch.zeros(2, 3, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 3, 2, dtype=torch.uint8)
    q, s = ActCheckpoint(codes, scales, BF16).matrices(codes.shape, codes.device, "linear")
    assert q.shape == (6, 64) and s.shape == (6, 2)
    off = torch.zeros(6 * 64 + 1, dtype=torch.uint8)[1:].view(torch.float8_e4m3fn).view(2, 3, 64)
    assert ActCheckpoint(off, scales, BF16).matrices(codes.shape, codes.device, "linear")[0].data_ptr() % 16 == 0
    for q, s, shape, text in ((codes, scales, (6, 64), "a checkpoint of shape"), (codes.to("meta"), scales, codes.shape, "on meta"),
                              (codes, scales.to("meta"), codes.shape, "scales on meta"), (codes, scales.int(), codes.shape, "uint8"),
                              (codes.half(), scales, codes.shape, "float8_e4m3fn"), (codes, scales[:, :2], codes.shape, "scales of shape"),
                              (codes, scales[..., :1], codes.shape, "scales of shape"), (codes[..., :48], scales, (2, 3, 48), "groups of 32")):
        with pytest.raises(ValueError, match=text):
            ActCheckpoint(q, s, BF16).matrices(torch.Size(shape), torch.device("cpu"), "linear")


P = 0x1000      # a pointer that no refused call follows


def _refused(rc, text):
    assert rc == -1 and text.encode() in _lib.load().mq_last_error(), (rc, _lib.load().mq_last_error())


def test_c_entry_of_the_dequantizer():
    f = _lib.load().mq_mxfp8_dequant
    _refused(f(P, P, P, 0, 4, 48, None), "divisible by 32")
    _refused(f(P, P, P, 7, 4, 64, None), "bad argument")
    _refused(f(P, P, P + 2, 0, 4, 64, None), "16 bytes")
    _refused(f(None, P, P, 0, 4, 64, None), "null pointer")
    assert f(None, None, None, 0, 0, 64, None) == 0


def test_c_entries_of_the_norms():
    lib = _lib.load()

    def forward(x=P, dtype=0, ldx=64, w=P, b=P, wdtype=0, y=P, xq=None, xs=None, yq=None, ys=None, rows=4, n=64, rms=0):
        return lib.mq_norm_forward(x, dtype, ldx, w, b, wdtype, y, xq, xs, yq, ys, P, P, rows, n, 1e-5, rms, None)

    _refused(forward(dtype=3), "bad argument")
    _refused(forward(rows=-1), "bad argument")
    _refused(forward(wdtype=1), "type")
    _refused(forward(ldx=63), "overlap")
    _refused(forward(x=None), "null pointer")
    _refused(forward(y=None), "null pointer")
    _refused(forward(xq=P), "null pointer")
    _refused(forward(yq=P, ys=P, n=48), "multiple of 32")
    _refused(forward(xq=P + 4, xs=P), "8 bytes")
    _refused(forward(rows=1 << 31), "too large")
    _refused(forward(rms=1), "no bias")
    _refused(forward(x=P + 2), "offsets")
    _refused(forward(ldx=66), "offsets")
    _refused(forward(x=P + 2, y=P + 2, yq=P, ys=P), "offsets")
    assert forward(rows=0, x=None, y=None) == 0

    def backward(dy=P, lddy=64, x=P, ldx=64, xs=None, mean=P, rstd=P, dw=P, db=P, ws=P, rows=4, n=64, rms=0):
        return lib.mq_norm_backward(dy, 0, lddy, x, ldx, xs, mean, rstd, P, 0, P, dw, db, ws, rows, n, rms, None)

    _refused(backward(lddy=10), "overlap")
    _refused(backward(ldx=10), "overlap")
    _refused(backward(mean=None), "null pointer")
    _refused(backward(rstd=None), "null pointer")
    _refused(backward(ws=None), "null pointer")
    _refused(backward(xs=P, n=48), "multiple of 32")
    _refused(backward(rms=1), "no bias")
    _refused(backward(dy=P + 2), "offsets")
    _refused(backward(lddy=65), "offsets")
    _refused(backward(xs=P, x=P + 8, lddy=66), "offsets")
    _refused(backward(xs=P, x=P + 4), "8-byte")
    assert backward(n=0, ws=P) == 0


def test_c_entries_of_the_linear_layers():
    lib = _lib.load()

    def forward(x=P, dtype=0, ldx=64, w=P, ldw=64, b=P, act=0, r=P, ldr=32, y=P, z=None, zq=None, zs=None, M=4, N=32, K=64, ws=P):
        return lib.mq_linear_forward(x, dtype, ldx, w, ldw, b, act, r, ldr, y, z, zq, zs, M, N, K, ws, None)

    _refused(forward(dtype=2), "bf16 or fp16")
    _refused(forward(act=5), "activation")
    _refused(forward(M=-1), "bad argument")
    _refused(forward(ldx=60), "overlap")
    _refused(forward(ldw=60), "overlap")
    _refused(forward(ldr=30), "overlap")
    _refused(forward(x=None), "null pointer")
    _refused(forward(y=None), "null pointer")
    _refused(forward(zq=P), "null pointer")
    _refused(forward(zq=P, zs=P, N=40, ldr=40), "multiple of 32")
    _refused(forward(zq=P + 2, zs=P), "4-byte")
    _refused(forward(K=1 << 31, ldx=1 << 31, ldw=1 << 31), "too large")
    assert forward(M=0) == 0 and forward(N=0) == 0

    size = ctypes.c_int64(-1)

    def workspace(product=0, a=P, lda=64, b=P, ldb=64, kept=0, M=4, N=32, K=64, out=ctypes.addressof(size)):
        return lib.mq_linear_workspace(product, a, lda, b, ldb, kept, M, N, K, out)

    _refused(workspace(product=3), "bad argument")
    _refused(workspace(out=None), "bad argument")
    _refused(workspace(lda=60), "overlap")
    for product in range(3):
        assert workspace(product, lda=8192, ldb=8192, M=300, N=512, K=8192) == 0 and size.value >= 0
    # a long sum over few outputs is cut, and then the partial sums need their memory; rows off 16 bytes are copied
    long = dict(M=48, N=512, K=8192)
    assert workspace(lda=8192, ldb=8192, **long) == 0 and size.value > 0
    partial = size.value
    assert workspace(a=P + 2, lda=8192, ldb=8192, **long) == 0 and size.value == partial + 48 * 8192 * 2
    assert workspace(lda=8192, ldb=8195, **long) == 0 and size.value == partial + 512 * 8192 * 2
    _refused(forward(**long, ldx=8192, ldw=8192, ldr=512, ws=None), "workspace")
    _refused(forward(**long, ldx=8192, ldw=8192, ldr=512, ws=P + 4), "workspace")

    def weight_grad(dz=P, lddz=32, x=P, ldx=64, xs=None, dw=P, M=4, N=32, K=64):
        return lib.mq_linear_weight_grad(dz, 0, lddz, x, ldx, xs, dw, M, N, K, P, None)

    _refused(weight_grad(lddz=31), "overlap")
    _refused(weight_grad(ldx=31), "overlap")
    _refused(weight_grad(dw=None), "null pointer")
    _refused(weight_grad(xs=P, K=48), "multiple of 32")
    _refused(weight_grad(xs=P, x=P + 8), "16-byte")
    _refused(lib.mq_linear_input_grad(P, 0, 32, None, 64, P, 4, 32, 64, P, None), "null pointer")
    _refused(lib.mq_linear_input_grad(P, 2, 32, P, 64, P, 4, 32, 64, P, None), "bf16 or fp16")

    def act_grad(dy=P, lddy=32, z=P, zs=None, act=1, db=P, ws=P, M=4, N=32):
        return lib.mq_activation_backward(dy, 0, lddy, z, zs, act, P, db, ws, M, N, None)

    _refused(act_grad(z=None), "null pointer")
    _refused(act_grad(ws=None), "null pointer")
    _refused(act_grad(act=-1), "activation")
    _refused(act_grad(zs=P, N=40, lddy=40), "multiple of 32")
    _refused(act_grad(lddy=31), "overlap")
