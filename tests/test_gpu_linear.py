"""Linear layers against the formulas in 64 bits.

Small whole numbers make every sum exact, so that the product's results have to be the rounded true ones to the last bit, whatever
the tile, the splits and the order.  With other numbers a sum of K products is off by at most K 2^-23 of the sum of their magnitudes
(fp32 additions in any order, each off by at most a step), and an activation, whose slope is at most 1.13, by that and 2^-20 more."""

import itertools

import pytest
import torch

from miles_amd import _lib
from miles_amd.kernels import linear as linear_module
from miles_amd.kernels.linear import linear
from miles_amd.kernels.norm import rms_norm
from miles_amd.kernels.quant.act_checkpoint import checkpoint_activation
from miles_amd.utils.mxfp8 import mxfp8_quantize
from tests.operator_checks import act64, f64, restored64, slope64, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16]
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _whole(g, *shape, dtype):
    return torch.randint(-2, 3, shape, generator=g).to(dtype).to(DEV)


SIZES = [(1, 64, 64), (1, 1, 1), (1, 2560, 4096), (2, 9, 5), (5, 128, 96), (16, 320, 2048), (17, 33, 45), (48, 512, 4096), (64, 2560, 640),
         (100, 40, 8), (129, 136, 72), (130, 264, 1000), (256, 512, 256), (257, 260, 130), (511, 777, 129), (700, 96, 3000), (1024, 2048, 512),
         (2048, 1024, 64), (3000, 64, 32), (2000, 2560, 640)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_whole_numbers_are_exact(m, n, k, dtype):
    g = torch.Generator().manual_seed(m + n + k)
    x, w, b, r = (_whole(g, *s, dtype=dtype).requires_grad_(True) for s in ((m, k), (n, k), (n,), (m, n)))
    dy = _whole(g, m, n, dtype=dtype)
    z = f64(x) @ f64(w).t()
    for act, bias, residual in ((None, None, None), (None, b, r), ("relu", b, None), ("relu", None, r)):
        zz = z + f64(bias) if bias is not None else z
        want = act64(zz, act) + (f64(r) if residual is not None else 0)
        leaves = [t for t in (x, w, bias, residual) if t is not None]
        dz = f64(dy) * slope64(zz, act)
        expect = [dz @ f64(w), dz.t() @ f64(x)] + ([dz.sum(0)] if bias is not None else []) + ([f64(dy)] if residual is not None else [])
        for checkpoint in (False, True) if k % 32 == 0 and n % 32 == 0 else (False,):
            y = linear(x, w, bias, activation=act, residual=residual, checkpoint=checkpoint)
            assert torch.equal(f64(y), f64(want.to(dtype))), (act, checkpoint)
            for got, e, name in zip(torch.autograd.grad(y, leaves, dy), expect, ("x", "w", "b", "r")):
                assert torch.equal(f64(got), f64(e.to(dtype))), (act, checkpoint, name)


def _random(m, n, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(dtype).to(DEV).requires_grad_(True)  # noqa: E731
    return make(m, k), make(n, k, scale=2 * k**-0.5), make(n, scale=0.5), make(m, n), make(m, n).detach()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 96, 256), (33, 160, 64), (300, 512, 224), (77, 65, 91), (40, 2048, 2048)])
def test_activations(m, n, k, act, dtype):
    x, w, b, r, dy = _random(m, n, k, dtype, seed=m)
    z = f64(x) @ f64(w).t() + f64(b)
    dz_sum = (k + 2) * 2.0**-23 * (f64(x).abs() @ f64(w).abs().t() + f64(b).abs())
    half = torch.finfo(dtype).eps / 2
    for checkpoint in (False, True) if k % 32 == 0 and n % 32 == 0 else (False,):
        y = linear(x, w, b, activation=act, residual=r, checkpoint=checkpoint)
        within(y, act64(z, act) + f64(r), 1.2 * dz_sum + 2.0**-20 * (z.abs() + f64(r).abs()), "y")
        grads = torch.autograd.grad(y, (x, w, b, r), dy)
        # what the layer kept, from a forward pass by itself
        _y, kept, scales = linear_module._forward(x.detach(), w.detach(), b.detach(), linear_module.ACTIVATIONS[act], None, act is not None, checkpoint)
        kx = restored64(*mxfp8_quantize(x.detach())) if checkpoint else f64(x)
        if act is None:
            dz, d_dz = f64(dy), torch.zeros_like(z)
        else:
            kz = restored64(kept, scales) if checkpoint else f64(kept)
            if checkpoint:
                scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.cpu().double() - 127).repeat_interleave(32, -1).to(DEV)
                assert ((kz - z).abs() <= 2.0**-4 * (z.abs() + dz_sum) + dz_sum + 2.0**-10 * scale).all()
            else:
                within(kept, z, dz_sum, "z")
            dz = f64(dy) * slope64(kz, act)
            # the slope's own 32-bit steps, and the rounding of dz on its way into the products
            d_dz = 2.0**-19 * f64(dy).abs() * (1 + kz.abs())
        order = lambda count: (count + 2) * 2.0**-23  # noqa: E731
        rounded = d_dz + (half * dz.abs() + 2.0**-25 if act is not None else 0)
        within(grads[0], dz @ f64(w), rounded @ f64(w).abs() + order(n) * (dz.abs() @ f64(w).abs()), "dx")
        within(grads[1], dz.t() @ kx, rounded.t() @ kx.abs() + order(m) * (dz.abs().t() @ kx.abs()), "dw")
        within(grads[2], dz.sum(0), d_dz.sum(0) + order(m) * dz.abs().sum(0), "db")
        assert torch.equal(grads[3], dy)


@pytest.mark.parametrize("act", ACTS[1:])
def test_slopes_against_differences(act):
    """The kernel's slopes at 4096 places against central differences of the activation in 64 bits (step 2^-12: off by 2^-24 of its
    third derivative, at most 2), away from the kink of relu."""
    z = torch.linspace(-9, 9, 4096, dtype=torch.float64).to(torch.bfloat16).view(1, -1).to(DEV)
    z = z[z.abs() > 2.0**-10].view(1, -1)
    n = z.shape[1]
    out = torch.empty_like(z)
    dy = torch.ones_like(z)
    _lib.check(_lib.load().mq_activation_backward(dy.data_ptr(), 0, n, z.data_ptr(), None, linear_module.ACTIVATIONS[act], out.data_ptr(), None, None, 1,
                                                  n, None))
    h = 2.0**-12
    want = (act64(f64(z) + h, act) - act64(f64(z) - h, act)) / (2 * h)
    within(out, want, torch.full_like(want, 2.0**-20 + 2.0**-22), act)


@pytest.mark.parametrize("dtype", TYPES)
def test_kept_z_is_the_quantizers(dtype):
    g = torch.Generator().manual_seed(2)
    for m, n, k in ((5, 64, 32), (300, 320, 200), (600, 1024, 512), (48, 512, 4096)):
        x, w, b = _whole(g, m, k, dtype=dtype), _whole(g, n, k, dtype=dtype), _whole(g, n, dtype=dtype)
        _y, codes, scales = linear_module._forward(x, w, b, 3, None, True, True)
        q, s = mxfp8_quantize((f64(x) @ f64(w).t() + f64(b)).float())       # whole numbers: z is exact
        assert torch.equal(codes.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scales, s)


def _in_nan(t, left, right):
    """t inside a larger matrix of NaN, its rows apart."""
    big = torch.full((t.shape[0] + 2, left + t.shape[1] + right), float("nan"), dtype=t.dtype, device=DEV)
    view = big[1:-1, left:left + t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("m,n,k", [(1, 40, 72), (3, 8, 8), (70, 136, 200), (260, 264, 104), (33, 7, 61), (300, 130, 333)])
@pytest.mark.parametrize("left,right", [(8, 16), (3, 2)])
def test_rows_apart_with_nan_between(m, n, k, left, right):
    """Whatever lies beyond a row's end, or behind the last row, does not reach the result: views on and off 16 bytes, and inner sizes that
    end inside a step."""
    g = torch.Generator().manual_seed(k)
    x0, w0, r0, dy0 = (_whole(g, *s, dtype=torch.bfloat16) for s in ((m, k), (n, k), (m, n), (m, n)))
    x, w, r, dy = (_in_nan(t, left, right) for t in (x0, w0, r0, dy0))
    for t in (x, w, r):
        t.requires_grad_(True)
    y = linear(x, w, residual=r)
    assert torch.equal(f64(y), f64((f64(x0) @ f64(w0).t() + f64(r0)).bfloat16()))
    gx, gw, gr = torch.autograd.grad(y, (x, w, r), dy)
    assert torch.equal(f64(gx), f64((f64(dy0) @ f64(w0)).bfloat16())) and torch.equal(f64(gw), f64((f64(dy0).t() @ f64(x0)).bfloat16()))
    assert torch.equal(gr, dy0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 7, 16])
@pytest.mark.parametrize("n,k", [(17, 1543), (33, 2048), (40, 1096), (16, 255), (1, 256), (15, 257), (160, 4104)])
def test_a_few_tokens_with_nan_around_their_rows(m, n, k, dtype):
    g = torch.Generator().manual_seed(m + k)
    x0, w0 = _whole(g, m, k, dtype=dtype), _whole(g, n, k, dtype=dtype)
    want = f64((f64(x0) @ f64(w0).t()).to(dtype))
    for left, right in ((0, 0), (8, 8 - k % 8), (3, 2), (1, 0)):
        assert torch.equal(f64(linear(_in_nan(x0, left, right), _in_nan(w0, left, right))), want), (left, right)
    assert torch.equal(f64(linear(x0, _in_nan(w0, 5, 0))), want)


def test_strides_and_shapes():
    g = torch.Generator().manual_seed(4)
    big, w = _whole(g, 4, 6, 96, dtype=torch.bfloat16), _whole(g, 40, 64, dtype=torch.bfloat16)
    for x, ww in ((big[..., 16:80], w), (big[:, ::2, 8:72], w), (big[0, 0, :64], w), (big.permute(1, 0, 2)[..., :64], w),
                  (big[:1, :1, :64].expand(4, 6, 64), w), (big[..., :64], _whole(g, 64, 40, dtype=torch.bfloat16).t()), (big[..., :40], w.t())):
        x, ww = x.detach().requires_grad_(True), ww.detach().requires_grad_(True)
        y = linear(x, ww)
        assert y.shape == (*x.shape[:-1], ww.shape[0])
        assert torch.equal(f64(y), f64((f64(x) @ f64(ww).t()).bfloat16()))
        gx, gw = torch.autograd.grad(y.float().sum(), (x, ww))          # the gradient has no memory of its own
        ones = torch.ones(y.shape, dtype=torch.float64, device=DEV)
        assert torch.equal(f64(gx), f64((ones @ f64(ww)).bfloat16()))
        assert torch.equal(f64(gw), f64((ones.reshape(-1, ww.shape[0]).t() @ f64(x).reshape(-1, x.shape[-1])).bfloat16()))


def test_empty_sizes():
    for m, n, k in ((0, 32, 64), (4, 0, 64), (4, 32, 0), (0, 0, 0)):
        for checkpoint in (False, True):
            x, w, b = (torch.ones(s, dtype=torch.bfloat16, device=DEV, requires_grad=True) for s in ((m, k), (n, k), (n,)))
            y = linear(x, w, b, activation="silu", checkpoint=checkpoint)
            want = torch.nn.functional.silu(torch.ones(m, n, dtype=torch.float64, device=DEV)) if k == 0 else torch.zeros(m, n, device=DEV)
            assert y.shape == (m, n) and (k != 0 or torch.equal(f64(y), f64(want.bfloat16())))
            gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
            assert gx.shape == x.shape and gw.shape == w.shape and (gw == 0).all() and (gx == 0).all() and (m or (gb == 0).all())


def test_special_values_stay_in_their_places():
    g = torch.Generator().manual_seed(6)
    x, w = _whole(g, 70, 96, dtype=torch.bfloat16), _whole(g, 130, 96, dtype=torch.bfloat16)
    clean = linear(x, w)
    x[3, 5], x[9, 0] = float("nan"), float("inf")
    w[:, 0] = 1
    clean = linear(x.nan_to_num(0, 0, 0), w)
    for act in ACTS:
        y = linear(x, w, activation=act)
        rest = [i for i in range(70) if i not in (3, 9)]
        assert y[3].isnan().all() and (y[9] == float("inf")).all()
        assert torch.equal(y[rest], linear(x[rest], w, activation=act))
    assert torch.equal(linear(x, w)[rest], clean[rest])


def test_one_copy_for_several_layers():
    x, w1, b, r, dy = _random(64, 96, 128, torch.bfloat16, seed=7)
    copy = checkpoint_activation(x)
    shared = linear(x, w1, b, activation="gelu", checkpoint=copy)
    own = linear(x, w1, b, activation="gelu", checkpoint=True)
    assert torch.equal(shared, own)
    for p, q in zip(torch.autograd.grad(shared, (x, w1, b), dy), torch.autograd.grad(own, (x, w1, b), dy)):
        assert torch.equal(p, q)
    # a misaligned copy is taken too
    raw = torch.empty(64 * 128 + 8, dtype=torch.uint8, device=DEV)[8:].view(64, 128)
    raw.copy_(copy.codes.view(torch.uint8))
    copy.codes = raw.view(torch.float8_e4m3fn)
    assert torch.equal(torch.autograd.grad(linear(x, w1, checkpoint=copy), w1, dy)[0], torch.autograd.grad(linear(x, w1, checkpoint=True), w1, dy)[0])


def test_only_what_asks_has_a_gradient():
    x, w, b, r, dy = _random(40, 64, 96, torch.bfloat16, seed=8)
    full = torch.autograd.grad(linear(x, w, b, activation="silu", residual=r, checkpoint=True), (x, w, b, r), dy)
    for wanted in itertools.product((False, True), repeat=4):
        if not any(wanted):
            continue
        args = [t if want else t.detach() for t, want in zip((x, w, b, r), wanted)]
        y = linear(args[0], args[1], args[2], activation="silu", residual=args[3], checkpoint=True)
        got = torch.autograd.grad(y, [t for t, want in zip(args, wanted) if want], dy)
        assert all(torch.equal(p, q) for p, q in zip(got, [t for t, want in zip(full, wanted) if want]))


def test_again_the_same_bits():
    for m, n, k in ((48, 512, 4096), (1, 2560, 2560), (700, 96, 3000)):
        x, w, b, r, dy = _random(m, n, k, torch.float16, seed=9)
        runs = []
        for _ in range(3):
            y = linear(x, w, b, activation="gelu", residual=r)
            runs.append([y, *torch.autograd.grad(y, (x, w, b), dy)])
        assert all(torch.equal(p, q) for run in runs[1:] for p, q in zip(run, runs[0]))


def test_offsets_beyond_32_bits():
    m, k, n = 330_000, 8192, 64
    x = torch.empty((m, k), dtype=torch.bfloat16, device=DEV)
    x.fill_(0)
    at = torch.tensor([0, 7, m // 2, m - 1], device=DEV)
    x[at, 0], x[at, k - 1] = 1, torch.tensor([1, 2, 3, 4], dtype=torch.bfloat16, device=DEV)
    w = torch.zeros((n, k), dtype=torch.bfloat16, device=DEV)
    w[:, 0], w[:, k - 1] = 8, 1
    w.requires_grad_(True), x.requires_grad_(True)
    y = linear(x, w)
    assert torch.equal(y[at, 0].float(), torch.tensor([9.0, 10, 11, 12], device=DEV)) and float(y.float().sum()) == 64 * 42
    dy = torch.zeros_like(y)
    dy[at] = 1
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    assert float(gw[:, 0].float().sum()) == 4 * n and float(gw[:, k - 1].float().sum()) == 10 * n and float(gw.float().sum()) == 14 * n
    assert (gx[at, 0] == 8 * n).all() and (gx[at, k - 1] == n).all() and float(gx.float().abs().sum()) == 4 * 9 * n


def test_captured_and_replayed():
    shapes = (300, 512, 1024)
    x, w, b, r, dy = _random(*shapes, torch.bfloat16, seed=11)

    def step():
        y = linear(x, w, b, activation="gelu", residual=r, checkpoint=True)
        small = linear(x[:1].detach(), w.detach(), b.detach())
        return [y.detach(), small, *torch.autograd.grad(y, (x, w, b, r), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(3):
        with torch.no_grad():
            for t, v in zip((x, w, b, r, dy), _random(*shapes, torch.bfloat16, seed=30 + seed)):
                t.copy_(v)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_two_streams_at_once():
    x, w, b, r, dy = _random(48, 512, 4096, torch.bfloat16, seed=12)
    want = [linear(x, w, b), *torch.autograd.grad(linear(x, w, b), (x, w), dy)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                y = linear(x, w, b)
                outs.append([y, *torch.autograd.grad(y, (x, w), dy)])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for out in outs for p, q in zip(out, want))


def test_a_norm_and_two_layers_in_8_bits():
    """The block as a training program runs it: the norm hands its 8-bit copy to the layers behind it, and every gradient is the formula's
    for the values that were kept."""
    m, h, f = 200, 256, 512
    x, w1, b1, _r, dy = _random(m, f, h, torch.bfloat16, seed=13)
    w2 = (torch.randn(h, f, generator=torch.Generator().manual_seed(1)) * f**-0.5).to(torch.bfloat16).to(DEV).requires_grad_(True)
    gamma = torch.ones(h, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    dy = dy[:, :h].contiguous()
    y, copy = rms_norm(x, gamma, checkpoint=True, output_checkpoint=True)
    a = linear(y, w1, b1, activation="silu", checkpoint=copy)
    out = linear(a, w2, residual=x, checkpoint=True)
    got = torch.autograd.grad(out, (x, gamma, w1, b1, w2), dy)
    # the same, layer by layer
    y1 = y.detach().requires_grad_(True)
    a1 = linear(y1, w1, b1, activation="silu", checkpoint=True)
    a2 = a1.detach().requires_grad_(True)
    out2 = linear(a2, w2, residual=x.detach(), checkpoint=True)
    assert torch.equal(out, out2)
    da, dw2 = torch.autograd.grad(out2, (a2, w2), dy)
    dy1, dw1, db1 = torch.autograd.grad(a1, (y1, w1, b1), da)
    dx, dgamma = torch.autograd.grad(rms_norm(x, gamma, checkpoint=True), (x, gamma), dy1)
    for p, q in zip(got, (dx + dy, dgamma, dw1, db1, dw2)):
        assert torch.equal(p, q)
    # what the 8-bit copies cost: the weights' gradients against those of copies that are not rounded
    plain = linear(linear(rms_norm(x, gamma), w1, b1, activation="silu"), w2, residual=x)
    assert torch.equal(plain, out)
    exact = torch.autograd.grad(plain, (x, gamma, w1, b1, w2), dy)
    for p, q in zip(got, exact):
        assert float((f64(p) - f64(q)).norm() / f64(q).norm()) < 2.0**-4


def test_refusals():
    x, w, b, r, _dy = _random(4, 64, 32, torch.bfloat16, seed=14)
    kept = checkpoint_activation(x)
    for call, text in ((lambda: linear(x.float(), w), "bfloat16 or float16"), (lambda: linear(x, w.half()), "weight is"),
                       (lambda: linear(x, w[:, :31]), "weight of shape"), (lambda: linear(x, w, b[:3]), "bias of shape"),
                       (lambda: linear(x, w, residual=r[:, :3]), "residual of shape"), (lambda: linear(x, w, b.float()), "bias is"),
                       (lambda: linear(x, w, activation="tanh"), "unknown activation"), (lambda: linear(x, w.cpu()), "weight on"),
                       (lambda: linear(x[:, :30], w[:, :30], checkpoint=True), "groups of 32"),
                       (lambda: linear(x, w[:40], activation="relu", checkpoint=True), "groups of 32"),
                       (lambda: linear(x[:2], w, checkpoint=kept), "a checkpoint of shape"), (lambda: linear(x, w, checkpoint=8), "ActCheckpoint")):
        with pytest.raises(ValueError, match=text):
            call()
    g = torch.autograd.grad(linear(x, w).float().square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_forward_mode_derivatives_are_refused():
    x, w, _b, _r, _dy = (t.detach() for t in _random(4, 64, 32, torch.bfloat16, seed=15))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: linear(dual, w), lambda: rms_norm(dual)):
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()
        assert torch.equal(linear(x, w), linear(x.clone(), w))


def test_native_and_python_host_layers_agree(monkeypatch):
    """An ordinary call makes its graph node in native code, any other in Python: the same bits, and only what asks has a gradient."""
    from miles_amd.kernels import norm as norm_mod
    from miles_amd.kernels.norm import layer_norm

    class Declines:
        def __getattr__(self, name):
            return lambda *args: None

    x, w, b, r, dy = _random(40, 64, 96, torch.bfloat16, seed=21)
    gamma, beta = (torch.randn(96, device=DEV).bfloat16().requires_grad_(True) for _ in range(2))

    def everything():
        out = []
        for wanted in itertools.product((False, True), repeat=3):
            if any(wanted):
                gx, gw, gb = (t if want else t.detach() for t, want in zip((x, gamma, beta), wanted))
                leaves = [t for t, want in zip((gx, gw, gb), wanted) if want]
                for ww, bb in ((gw, gb), (gw, None), (None, gb), (None, None)):
                    for kw in ({}, {"checkpoint": True}):
                        y = layer_norm(gx.view(8, 5, 96), ww, bb, **kw)
                        if y.requires_grad:
                            out.append(y.detach())
                            out.extend(g for g in torch.autograd.grad(y.sum(0), leaves, dy[:5, :1].expand(5, 96), allow_unused=True) if g is not None)
        for wanted in itertools.product((False, True), repeat=4):
            if any(wanted):
                args = [t if want else t.detach() for t, want in zip((x, w, b, r), wanted)]
                for bias, residual in itertools.product((args[2], None), (args[3], None)):
                    for kw in ({}, {"checkpoint": True}, {"checkpoint": checkpoint_activation(x)}):
                        for act in (None, "silu"):
                            y = linear(args[0], args[1], bias, activation=act, residual=residual, **kw)
                            if y.requires_grad:
                                out.append(y.detach())
                                leaves = [t for t, want in zip(args, wanted) if want]
                                out.extend(g for g in torch.autograd.grad(y, leaves, dy, allow_unused=True) if g is not None)
        copy = checkpoint_activation(x)
        return out + [copy.codes.view(torch.uint8), copy.scales, copy.restore()]

    ours = everything()
    for module in (linear_module, norm_mod):
        monkeypatch.setattr(module, "native", Declines())
    monkeypatch.setattr("miles_amd.kernels.quant.act_checkpoint.native", Declines())
    monkeypatch.setattr("miles_amd.utils.mxfp8.native", Declines())
    theirs = everything()
    assert len(ours) == len(theirs) > 100 and all(torch.equal(p, q) for p, q in zip(ours, theirs))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_under_every_scale_in_the_weight_gradient(dtype):
    """dW of one-hot gradients is the kept input itself: every code under every exponent, as the layer's dtype holds it."""
    m, k = 255, 256 * 32
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat_interleave(32).repeat(m, 1)
    scales = torch.arange(m, dtype=torch.uint8, device=DEV).unsqueeze(1).expand(m, k // 32).contiguous()
    nan = (codes & 0x7F) == 0x7F
    codes[nan] = 0                                          # (a NaN would reach every row of its column)
    dz = torch.eye(m, dtype=dtype, device=DEV)
    dz8 = torch.zeros(m, 256, dtype=dtype, device=DEV)      # (columns a multiple of eight)
    dz8[:, :m] = dz
    for g, n in ((dz, m), (dz8, 256)):
        dw = torch.empty(n, k, dtype=dtype, device=DEV)
        ws = linear_module._workspace(2, g, codes, True, m, n, k)
        _lib.check(_lib.load().mq_linear_weight_grad(g.data_ptr(), _lib.DTYPE_CODE[dtype], n, codes.data_ptr(), k, scales.data_ptr(), dw.data_ptr(), m, n, k,
                                                     None if ws is None else ws.data_ptr(), None))
        kept = restored64(codes.view(torch.float8_e4m3fn).cpu(), scales.cpu())
        kept = (kept.clamp(-65504, 65504) if dtype == torch.float16 else kept).to(dtype)
        want = dz.double().cpu().t() @ kept.double()        # (a value that bf16 holds as an infinity makes its column NaN, 0 times it)
        got = dw[:m].double().cpu()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0, 1, 2), want.nan_to_num(0, 1, 2))
