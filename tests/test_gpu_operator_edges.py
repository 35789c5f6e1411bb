"""Norms and linear layers at the ends of their ranges: types that are mixed, arguments far out, rows without any spread."""

import pytest
import torch

from miles_amd import _lib
from miles_amd.kernels.linear import ACTIVATIONS, linear
from miles_amd.kernels.norm import layer_norm, rms_norm
from miles_amd.kernels.quant.act_checkpoint import ActCheckpoint, checkpoint_activation
from tests.operator_checks import f64, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALVES = [torch.bfloat16, torch.float16]


def _off(t):
    """t at an address that is no multiple of 16, its rows apart: what the native host layer leaves to Python."""
    big = torch.zeros(t.shape[0], t.shape[1] + 8, dtype=t.dtype, device=DEV)
    view = big[:, 3:3 + t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("place", [torch.Tensor.contiguous, _off], ids=["contiguous", "off"])
def test_the_gradient_of_an_fp32_bias_without_a_weight_is_fp32(place, dtype):
    """Sums of 100 rows, at most 100 2^-24 of the magnitudes off before the rounding to fp32; the largest is beyond fp16."""
    g = torch.Generator().manual_seed(1)
    x, dy = (place(torch.randn((100, 96), generator=g).to(dtype).to(DEV)) for _ in range(2))
    dy[:, 5] = 1000.0
    b = torch.randn(96, generator=g).to(DEV).requires_grad_(True)
    db = torch.autograd.grad(layer_norm(x, None, b), b, dy)[0]
    assert db.dtype == torch.float32 and db[5] == 100_000
    within(db, f64(dy).sum(0), 100 * 2.0**-24 * f64(dy).abs().sum(0), "db")


# magnitudes from where every activation is saturated in fp32 up to the types' largest finite values
FAR = {torch.bfloat16: [20.0, 1e3, 65504.0, 1e10, 2e13, 1e19, 2e19, 1e30, torch.finfo(torch.bfloat16).max], torch.float16: [20.0, 1e3, 4096.0, 65504.0]}


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", [a for a in ACTIVATIONS if a])
def test_arguments_far_out(act, dtype):
    """There an activation is its argument or 0, and its slope 1 or 0 (the nearest place, -20, is 2e-9 of them off in SiLU, whose values
    are -20 e^-20 and less); one NaN would take a row of dx and one of dW with it."""
    far = torch.tensor(FAR[dtype], dtype=dtype, device=DEV)
    z = torch.cat([far, -far])
    n, k = z.numel(), 32
    x, dy = torch.zeros(3, k, dtype=dtype, device=DEV).requires_grad_(True), torch.ones(3, n, dtype=dtype, device=DEV)
    w, b = torch.eye(n, k, dtype=dtype, device=DEV).requires_grad_(True), z.clone().requires_grad_(True)
    y = linear(x, w, b, activation=act)
    on = (z > 0).double()
    assert (f64(y) - f64(z) * on).abs().max() <= 2.0**-24
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (f64(db) - 3 * on).abs().max() <= 2.0**-22 and (f64(dx) - (f64(dy) * on) @ f64(w)).abs().max() <= 2.0**-23 and (dw == 0).all()
    # from 16-bit and from 8-bit copies alike
    pad = torch.cat([z, torch.zeros(-n % 32, dtype=dtype, device=DEV)])
    x, b = torch.zeros(3, k, dtype=dtype, device=DEV), pad.clone().requires_grad_(True)
    y = linear(x, torch.zeros(pad.numel(), k, dtype=dtype, device=DEV), b, activation=act, checkpoint=True)
    db = torch.autograd.grad(y, b, torch.ones_like(y))[0]
    assert db.isfinite().all() and ((db[:n] == 3) | (db[:n] == 0) | (z.abs() < far.max() * 2.0**-8)).all()
    assert (db[:n][z == far.max()] == 3).all() and (db[:n][z == -far.max()] == 0).all()      # (bf16: kept as infinities)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows", [3, 40])
def test_small_values_of_gelu_keep_their_bits(rows, dtype):
    """Down to where bf16 results are subnormal: Phi is claimed to 5e-5 of itself below -3 and to 2.5e-7 everywhere; 16 steps of fp32 (up to
    84 of them in the exponent's product) and half a step of the result come on top."""
    z = torch.linspace(-12.75, 1, 4096, dtype=torch.float64).to(dtype).to(DEV)
    phi, bell = torch.special.erfc(f64(z) * -(0.5**0.5)) / 2, torch.exp(-f64(z).square() / 2) / (2 * torch.pi) ** 0.5
    off = torch.where(f64(z) < -3, 5e-5 * phi, torch.full_like(phi, 2.5e-7)) + (16 + f64(z).square()) * 2.0**-24 * phi
    half, smallest = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x, w = torch.zeros(rows, 32, dtype=dtype, device=DEV), torch.zeros(4096, 32, dtype=dtype, device=DEV)
    y = f64(linear(x, w, z, activation="gelu"))
    want = f64(z) * phi
    assert ((y - want).abs() <= half * want.abs() + 1.01 * f64(z).abs() * off + smallest / 2).all()
    assert (y == y[0]).all()
    slopes = torch.empty_like(z)
    _lib.check(_lib.load().mq_activation_backward(torch.ones_like(z).data_ptr(), _lib.DTYPE_CODE[dtype], 4096, z.data_ptr(), None, ACTIVATIONS["gelu"],
                                                  slopes.data_ptr(), None, None, 1, 4096, None))
    want = phi + f64(z) * bell
    off += (16 + f64(z).square()) * 2.0**-24 * f64(z).abs() * bell
    assert ((f64(slopes) - want).abs() <= half * want.abs() + 1.01 * off + smallest / 2).all()


def test_scales_of_another_shape_are_refused_whatever_their_number():
    x = torch.randn(6, 4, 64, device=DEV).bfloat16().requires_grad_(True)
    w = torch.randn(32, 64, device=DEV).bfloat16().requires_grad_(True)
    kept = checkpoint_activation(x)
    for scales in (kept.scales.reshape(4, 6, 2), kept.scales.reshape(24, 2), kept.scales.reshape(6, 8), kept.scales.unsqueeze(0)):
        for arg in (x, x.detach()):
            with pytest.raises(ValueError, match="scales of shape"):
                linear(arg, w, checkpoint=ActCheckpoint(kept.codes, scales, x.dtype))
    assert linear(x, w, checkpoint=kept).shape == (6, 4, 32)


@pytest.mark.parametrize("dtype", [*HALVES, torch.float32])
@pytest.mark.parametrize("n", [1, 40, 96, 1000, 2560, 2563, 7168, 33000])
def test_a_row_of_one_value_has_no_spread(n, dtype):
    """Sums of n times 1000 or -3.5 are exact below 2^24 quanta, their quotients by n too: xhat is 0 and with it everything that it is a factor of.
    What is left of dx, rstd (g - mean g), is off by 2^-18 of the magnitudes as all of the norms' sums are."""
    g = torch.Generator().manual_seed(n)
    x = torch.empty(9, n, dtype=dtype, device=DEV)
    x[::2], x[1::2] = 1000.0, -3.5
    w, b = ((torch.randn(n, generator=g)).to(dtype).to(DEV).requires_grad_(True) for _ in range(2))
    dy = torch.randn((9, n), generator=g).to(dtype).to(DEV)
    for place in (torch.Tensor.contiguous, _off):
        leaf = place(x).requires_grad_(True)
        y = layer_norm(leaf, w, b, 1e-5)
        dx, dw, db = torch.autograd.grad(y, (leaf, w, b), dy)
        assert torch.equal(y, b.detach().expand(9, n)) and (dw == 0).all()
        grads = f64(dy) * f64(w)
        rstd = 1e5**0.5
        within(dx, rstd * (grads - grads.mean(1, keepdim=True)), 4 * rstd * 2.0**-18 * (grads.abs() + grads.abs().mean(1, keepdim=True)), "dx")


@pytest.mark.parametrize("n,rows", [(4, (1 << 26) + 9), (5, (1 << 26) + 9), (1032, (1 << 21) + 77)])
def test_rows_beyond_one_launch(n, rows):
    """More rows than a launch has lanes for; each has the bits that it has in a short tensor."""
    x = torch.empty((rows, n), dtype=torch.bfloat16, device=DEV)
    x.view(torch.int16).random_(0x3C00, 0x4000)
    w, b = (torch.randn(n, device=DEV).bfloat16().requires_grad_(True) for _ in range(2))
    x.requires_grad_(True)
    for call in (lambda t: layer_norm(t, w, b), lambda t: rms_norm(t, w)):
        y = call(x)
        dx = torch.autograd.grad(y, x, y.detach())[0]
        for at in (0, 1 << 20, (1 << 21) - 16, 1 << 21, (1 << 25) - 16, 1 << 26, rows - 32):
            at = min(at, rows - 32) // 8 * 8
            part = x[at:at + 32].detach().requires_grad_(True)
            want = call(part)
            assert torch.equal(y[at:at + 32], want), at
            assert torch.equal(dx[at:at + 32], torch.autograd.grad(want, part, want.detach())[0]), at
        del y, dx


def test_8_bit_copies_of_rows_beyond_one_launch():
    rows, n = (1 << 25) + 41, 32
    x = torch.empty((rows, n), dtype=torch.bfloat16, device=DEV)
    x.view(torch.int16).random_(0x3C00, 0x4000)
    x.requires_grad_(True)
    y, copy = rms_norm(x, checkpoint=True, output_checkpoint=True)
    dx = torch.autograd.grad(y, x, y.detach())[0]
    for at in (0, (1 << 25) - 16, rows // 8 * 8 - 32):
        part = x[at:at + 32].detach().requires_grad_(True)
        want, kept = rms_norm(part, checkpoint=True, output_checkpoint=True)
        assert torch.equal(copy.codes[at:at + 32].view(torch.uint8), kept.codes.view(torch.uint8)) and torch.equal(copy.scales[at:at + 32], kept.scales)
        assert torch.equal(dx[at:at + 32], torch.autograd.grad(want, part, want.detach())[0])


@pytest.mark.parametrize("dtype,small,large", [(torch.float16, 2.0**-24, 8.0), (torch.bfloat16, 2.0**-133, 2.0**20)])
@pytest.mark.parametrize("m,n,k", [(3, 64, 64), (40, 64, 64), (300, 512, 256), (1024, 2048, 512)])
def test_subnormal_operands_count(m, n, k, dtype, small, large):
    """Whole multiples of the smallest subnormal: exact sums, as with any whole numbers."""
    g = torch.Generator().manual_seed(k)
    x = (torch.randint(-3, 4, (m, k), generator=g).double() * small).to(dtype).to(DEV).requires_grad_(True)
    w = (torch.randint(-2, 3, (n, k), generator=g).double() * large).to(dtype).to(DEV).requires_grad_(True)
    y = linear(x, w)
    assert torch.equal(f64(y), f64((f64(x) @ f64(w).t()).to(dtype)))
    dw = torch.autograd.grad(y, w, torch.ones_like(y))[0]
    assert torch.equal(f64(dw), f64(f64(x).sum(0).expand(n, k).to(dtype)))


def test_a_residual_that_is_the_input():
    x, w = (torch.randn(s, 96, device=DEV).bfloat16().requires_grad_(True) for s in (40, 96))
    y = linear(x, w, residual=x)
    dy = torch.randn_like(y)
    before = dy.clone()
    dx = torch.autograd.grad(y, x, dy)[0]
    apart = x.detach().clone().requires_grad_(True)
    through = torch.autograd.grad(linear(apart, w, residual=x.detach()), apart, dy)[0]
    assert torch.equal(dx, through + dy) and torch.equal(dy, before)
