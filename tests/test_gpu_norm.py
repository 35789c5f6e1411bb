"""Layer norm and RMS norm against the formulas in 64 bits.

Before its rounding a result is off by what 32-bit sums are: a lane adds at most 40 numbers one behind the other, then at most 14
sums of lanes follow, so a sum is off by at most 64 2^-24 = 2^-18 of the sum of the magnitudes.  The bounds below carry that through the
formulas: the mean is off by 2^-18 mean|x|, 1/sigma relatively by 2^-18 and by that mean's part, which is second order."""

import pytest
import torch

from miles_amd.kernels import norm as norm_module
from miles_amd.kernels.norm import layer_norm, rms_norm
from miles_amd.utils.mxfp8 import mxfp8_quantize
from tests.operator_checks import f64, restored64, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0**-18


def _inputs(m, n, dtype, wdtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((m, n), generator=g) * torch.exp(torch.randn((m, 1), generator=g)) + 0.25).to(dtype).to(DEV)
    w = (1 + 0.2 * torch.randn(n, generator=g)).to(wdtype or dtype).to(DEV)
    b = (0.2 * torch.randn(n, generator=g)).to(wdtype or dtype).to(DEV)
    dy = torch.randn((m, n), generator=g).to(dtype).to(DEV)
    return x, w, b, dy


def _statistics(x, rms, eps):
    x = f64(x)
    mean = torch.zeros_like(x[:, :1]) if rms else x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    xhat = (x - mean) * rstd
    # what xhat may be off by
    return rstd, xhat, 2 * U * (xhat.abs() + (0 if rms else 1) * x.abs().mean(1, keepdim=True) * rstd)


def _check(x, w, b, dy, y, grads, rms, eps, kept=None):
    """y and (dx, dw, db) against the formulas; kept: the 8-bit xhat that the backward pass had."""
    rstd, xhat, dxhat = _statistics(x, rms, eps)
    w64 = f64(w) if w is not None else torch.ones(x.shape[1], dtype=torch.float64, device=DEV)
    b64 = f64(b) if b is not None else torch.zeros_like(w64)
    within(y, xhat * w64 + b64, dxhat * w64.abs() + U * (xhat * w64).abs() + U * b64.abs(), "y")
    if grads is None:
        return
    if kept is not None:
        xhat, dxhat = kept, torch.zeros_like(dxhat)
    dx, dw, db = grads
    d = f64(dy)
    g = d * w64
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    along = mean(g * xhat)
    flat = torch.zeros_like(along) if rms else mean(g)
    if dx is not None:
        slack = 4 * U * (g.abs() + mean(g.abs()) + xhat.abs() * mean((g * xhat).abs()))
        slack += dxhat * along.abs() + xhat.abs() * mean(g.abs() * dxhat)
        within(dx, rstd * (g - flat - xhat * along), rstd * slack, "dx")
    rows = x.shape[0]
    # a workgroup adds its rows one behind the other, then their sums come together
    order = (rows / 256 + 64) * 2.0**-24
    if dw is not None:
        within(dw, (d * xhat).sum(0), order * (d * xhat).abs().sum(0) + (d.abs() * dxhat).sum(0), "dw")
    if db is not None:
        within(db, d.sum(0), order * d.abs().sum(0), "db")


def _run(kind, x, w, b, eps, **kw):
    return rms_norm(x, w, eps, **kw) if kind == "rms" else layer_norm(x, w, b, eps, **kw)


WIDTHS = [1, 7, 33, 64, 512, 520, 1000, 1024, 2047, 2560, 4096, 7168, 8200, 16384, 20000, 33000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_forward_and_backward(kind, n, dtype):
    m = 5 if n > 8000 else 67
    x, w, b, dy = _inputs(m, n, dtype, seed=n)
    leaves = [t.requires_grad_(True) for t in ([x, w, b] if kind == "layer" else [x, w])]
    y = _run(kind, x, w, b, 1e-5)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(y, _run(kind, x, w, b, 1e-5))
    _check(x, w, b if kind == "layer" else None, dy, y, (*grads, None)[:3], kind == "rms", 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(1, 32), (33, 64), (4100, 96), (3, 512), (40, 2560), (1100, 4096), (9, 8192), (2, 16384), (3, 40960)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_kept_in_8_bits(kind, m, n, dtype):
    x, w, b, dy = _inputs(m, n, dtype, seed=m)
    rms = kind == "rms"
    # the codes that a norm of this input keeps
    codes, scales = norm_module._forward(x, w, None if rms else b, 1e-5, rms, True, True, False)[3:5]
    kept = restored64(codes, scales)
    _rstd, xhat, dxhat = _statistics(x, rms, 1e-5)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.cpu().double() - 127).repeat_interleave(32, -1).to(DEV)
    assert ((kept - xhat).abs() <= 2.0**-4 * (xhat.abs() + dxhat) + dxhat + 2.0**-10 * scale).all()
    assert (scale * 448 * (1 + 2.0**-20) >= xhat.abs()).all() and (scale > 0).all()
    leaves = [t.requires_grad_(True) for t in ([x, w] if rms else [x, w, b])]
    y = _run(kind, x, w, b, 1e-5, checkpoint=True)
    grads = torch.autograd.grad(y, leaves, dy)
    _check(x, w, None if rms else b, dy, y, (*grads, None)[:3], rms, 1e-5, kept)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [64, 2560, 8192, 40960])
def test_the_copy_of_the_result(n, dtype):
    x, w, b, dy = _inputs(13, n, dtype, seed=5)
    for grad in (False, True):
        x.requires_grad_(grad)
        y, copy = layer_norm(x.view(13, 1, n), w, b, output_checkpoint=True)
        q, s = mxfp8_quantize(y.detach())
        assert y.requires_grad == grad and not copy.codes.requires_grad and copy.shape == y.shape and copy.dtype == dtype
        assert torch.equal(copy.codes.view(torch.uint8), q.view(torch.uint8)) and torch.equal(copy.scales, s)
        assert torch.equal(y.view(13, n), layer_norm(x, w, b))
    gx = torch.autograd.grad(layer_norm(x, w, b, output_checkpoint=True)[0], x, dy)[0]
    assert torch.equal(gx, torch.autograd.grad(layer_norm(x, w, b), x, dy)[0])


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("n", [40, 2563, 33000])
def test_weights_in_fp32(n, dtype, wdtype):
    x, w, b, dy = _inputs(21, n, dtype, wdtype, seed=7)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(x, w, b, 1e-5)
    grads = torch.autograd.grad(y, leaves, dy)
    assert [g.dtype for g in grads] == [dtype, wdtype, wdtype]
    _check(x, w, b, dy, y, grads, False, 1e-5)


def test_without_weight_or_bias():
    x, w, b, dy = _inputs(9, 100, torch.bfloat16, seed=8)
    x.requires_grad_(True), b.requires_grad_(True), w.requires_grad_(True)
    for ww, bb in ((None, None), (w, None), (None, b)):
        y = layer_norm(x, ww, bb)
        grads = torch.autograd.grad(y, [t for t in (x, ww, bb) if t is not None], dy)
        _check(x, ww, bb, dy, y, (grads[0], grads[1] if ww is not None else None, grads[-1] if bb is not None else None), False, 1e-5)
    # only what asks for a gradient has one
    y = layer_norm(x.detach(), w, b.detach())
    _check(x, w, b, dy, y, (None, torch.autograd.grad(y, w, dy)[0], None), False, 1e-5)


def test_rows_more_than_the_partial_sums():
    for m, n in ((9000, 24), (2500, 1032)):
        x, w, b, dy = _inputs(m, n, torch.float32, seed=9)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        y = layer_norm(x, w, b)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        _check(x, w, b, dy, y, first, False, 1e-5)
        assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, leaves, dy)))     # and again the same bits


def test_strides_and_shapes():
    g = torch.Generator().manual_seed(3)
    big = torch.randn((50, 300), generator=g).to(torch.bfloat16).to(DEV)
    w = torch.ones(96, dtype=torch.bfloat16, device=DEV)
    for x in (big[:, 8:104], big[:, 3:99], big.t()[:96].t(), big[:48].view(6, 8, 300)[:, ::2, 5:101], big[:1, :96].expand(20, 96), big[0, :96]):
        for checkpoint in (False, True):
            leaf = x.detach().requires_grad_(True)
            y = layer_norm(leaf, w, checkpoint=checkpoint)
            assert y.shape == x.shape
            flat = x.reshape(-1, 96).contiguous().requires_grad_(True)
            want = layer_norm(flat, w, checkpoint=checkpoint)
            assert torch.equal(y.reshape(-1, 96), want)
            # a gradient that is one number everywhere, without memory of its own
            assert torch.equal(torch.autograd.grad(y.sum(), leaf)[0].reshape(-1, 96), torch.autograd.grad(want.sum(), flat)[0])


def test_empty_and_special_rows():
    w = torch.ones(64, dtype=torch.float32, device=DEV, requires_grad=True)
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    for checkpoint in (False, True):
        y = layer_norm(x, w, checkpoint=checkpoint)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == gx.shape == (0, 64) and (gw == 0).all()
    assert layer_norm(torch.empty(5, 0, device=DEV)).shape == (5, 0)
    x = torch.randn(6, 64, device=DEV)
    x[1], x[2, 5], x[3, 7], x[4] = 2.5, float("nan"), float("inf"), 0.0
    for checkpoint in (False, True):
        leaf = x.clone().requires_grad_(True)
        y = layer_norm(leaf, w, eps=1e-6, checkpoint=checkpoint)
        assert (y[1] == 0).all() and (y[4] == 0).all() and y[2].isnan().all() and y[3].isnan().any()
        clean = layer_norm(x[[0, 5]], w, eps=1e-6)
        assert torch.equal(y[[0, 5]], clean)
        dx = torch.autograd.grad(y, leaf, torch.ones_like(y))[0]
        assert dx[[0, 1, 4, 5]].isfinite().all()


def test_offsets_beyond_32_bits():
    m, n = 330_000, 8192                                   # 5.4 GB of bf16
    x = torch.empty((m, n), dtype=torch.bfloat16, device=DEV)
    x.view(torch.int16).random_(0x3C00, 0x4000)
    at = torch.tensor([0, 1, m // 2, m - 1], device=DEV)
    y = rms_norm(x)
    within(y[at], f64(x[at]) / torch.sqrt(f64(x[at]).square().mean(1, keepdim=True) + 1e-6), 4 * U * 8, "y")
    x.requires_grad_(True)
    dx = torch.autograd.grad(rms_norm(x), x, y)[0]
    few = x[at].detach().requires_grad_(True)
    assert torch.equal(dx[at], torch.autograd.grad(rms_norm(few), few, y[at])[0])


def test_against_differences():
    """fp32: the gradient along a direction against the difference of two forward passes.  The loss is a sum of 6 x 96 products; with a
    step of 2^-7 its third-order term is about 2^-14 of the second difference scale, below the 1 % asked for."""
    x, w, b, dy = _inputs(6, 96, torch.float32, seed=11)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(x, w, b), leaves, dy)
    g = torch.Generator().manual_seed(12)
    for i, grad in enumerate(grads):
        direction = torch.sign(grad) * (1 + torch.rand(grad.shape, generator=g).to(DEV)) * leaves[i].detach().abs().mean()
        h = 2.0**-7
        with torch.no_grad():
            moved = [[t + (s * h * direction if j == i else 0) for j, t in enumerate(leaves)] for s in (1, -1)]
            up, down = (float((f64(layer_norm(*p)) * f64(dy)).sum()) for p in moved)
        along = float((f64(grad) * f64(direction)).sum())
        assert abs((up - down) / (2 * h) - along) <= 0.01 * abs(along), (i, up, down, along)


def test_captured_and_replayed():
    x, w, b, dy = _inputs(300, 1024, torch.bfloat16, seed=13)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layer_norm(x, w, b, checkpoint=True)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]      # (no graph of these leaves outlives the step)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                     # two graphs of one step, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(3):
        fresh = _inputs(300, 1024, torch.bfloat16, seed=20 + seed)
        with torch.no_grad():
            for t, v in zip((x, w, b, dy), fresh):
                t.copy_(v)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_on_another_stream():
    x, w, b, dy = _inputs(2000, 2048, torch.bfloat16, seed=14)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(x, w, b), leaves, dy)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = torch.autograd.grad(layer_norm(x, w, b), leaves, dy)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals():
    x = torch.zeros(4, 40, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(40, dtype=torch.bfloat16, device=DEV)
    for call, text in ((lambda: layer_norm(x, w[:39]), "weight of shape"), (lambda: layer_norm(x, w.half()), "input's type"),
                       (lambda: layer_norm(x, w, w.float()), "weight is"), (lambda: layer_norm(x, w.cpu()), "the input on"),
                       (lambda: rms_norm(x, w, checkpoint=True), "groups of 32"), (lambda: rms_norm(x, output_checkpoint=True), "groups of 32"),
                       (lambda: layer_norm(torch.zeros((), device=DEV)), "at least one dimension")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(Exception, match="unsupported dtype"):
        layer_norm(x.double())
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    g = torch.autograd.grad(rms_norm(x).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
