"""Rotary positions against the formula in 64 bits, forward and backward."""

import pytest
import torch

from miles_amd import _lib
from miles_amd.kernels.rotary import rotary, rotary_frequencies
from tests.operator_checks import f64, within
from tests.serving_checks import DEV, turned64

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(*shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _check(x, y, *args, **kw):
    want, off = turned64(x, *args, **kw)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    within(y, want, off, "turned")
    rest = 2 * args[1].shape[0]
    assert torch.equal(y[..., rest:], x[..., rest:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,turned", [(2, 2), (8, 8), (64, 64), (80, 80), (96, 32), (128, 128), (128, 64), (192, 64), (256, 256), (67, 10), (130, 130), (1024, 1024), (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
def test_turned(interleaved, dim, turned, dtype):
    tokens = 37
    q, k = _randn(tokens, 6, dim, dtype=dtype), _randn(tokens, 2, dim, dtype=dtype, seed=1)
    freq = rotary_frequencies(turned, device=DEV)[0] if turned else torch.empty(0, dtype=torch.float64, device=DEV)
    positions = torch.arange(tokens, device=DEV) * 977 + 3
    y, z = rotary(q, k, positions, freq, interleaved=interleaved, scale=1.25)
    for x, got in ((q, y), (k, z)):
        _check(x, got, positions, freq, 1.25, interleaved)
    assert torch.equal(rotary(q, None, positions, freq, interleaved=interleaved, scale=1.25), y)
    # as views of a fused projection, at any address
    fused = torch.zeros(tokens, 8 * dim + 5, dtype=dtype, device=DEV)
    for off in (0, 3):
        a, b = fused[:, off:off + 6 * dim].view(tokens, 6, dim), fused[:, off + 6 * dim:off + 8 * dim].view(tokens, 2, dim)
        a.copy_(q), b.copy_(k)
        y2, z2 = rotary(a, b, positions, freq, interleaved=interleaved, scale=1.25)
        assert torch.equal(y2, y) and torch.equal(z2, z)
    # and back
    _check(y, rotary(y, None, positions, freq, interleaved=interleaved, inverse=True), positions, freq, 1.0, interleaved, True)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32])
@pytest.mark.parametrize("freq_type", [torch.float64, torch.float32])
def test_far_and_negative_positions(kind, freq_type):
    positions = torch.tensor([0, 1, -1, 4095, -4096, 1 << 20, (1 << 31) - 1, -(1 << 31), 123456789], dtype=kind, device=DEV)
    if kind == torch.int64:
        positions = torch.cat([positions, torch.tensor([1 << 40, -(1 << 45) + 1, 3 << 33], device=DEV)])
    freq = rotary_frequencies(128, 1e6, device=DEV)[0].to(freq_type)
    freq[1] = 7.25                                         # several turns from one position to the next
    x = _randn(len(positions), 3, 128, dtype=torch.float32)
    # an angle of 2^45 radians has 2^-8 of one in its last bit in 64 bits: the definition is that angle
    _check(x, rotary(x, None, positions, freq), positions, freq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 3, 513, 5000])
def test_tokens_of_a_batch(tokens, dtype):
    """Batches with positions of their own, with the same ones, with leading dimensions and orders of other kinds."""
    freq = rotary_frequencies(64, device=DEV)[0]
    x = _randn(2, tokens, 3, 64, dtype=dtype)
    own = torch.randint(0, 100000, (2, tokens), generator=torch.Generator().manual_seed(3)).to(DEV)
    one = own[0].contiguous()
    for positions in (own, one, one[None], own[:, :1], own.t().contiguous().t()):
        y = rotary(x, None, positions, freq)
        _check(x, y, positions.expand(2, tokens), freq)
        by_head = x.transpose(1, 2).contiguous().transpose(1, 2)             # [batch, heads, tokens, dim] in memory
        assert torch.equal(rotary(by_head, None, positions, freq), y)
        assert torch.equal(rotary(x[:, None], None, positions[:, None] if positions.dim() == 2 else positions, freq)[:, 0], y)
    assert torch.equal(rotary(x[0, 0], None, own[0, 0], freq), rotary(x, None, own, freq)[0, 0])
    assert torch.equal(rotary(x.flip(3).flip(3), None, own, freq), rotary(x, None, own, freq))
    assert rotary(x[:, :0], None, own[:, :0], freq).shape == (2, 0, 3, 64)
    wide = x[:, :, :1].expand(2, tokens, 5, 64)
    assert torch.equal(rotary(wide, None, own, freq), rotary(wide.contiguous(), None, own, freq))


def test_non_finite_values_stay_in_their_pairs():
    x = _randn(4, 2, 64, dtype=torch.bfloat16)
    x[0, 0, 5], x[1, 1, 40], x[2, 0, 63] = float("nan"), float("inf"), float("-inf")
    freq = rotary_frequencies(64, device=DEV)[0]
    positions = torch.arange(1, 5, device=DEV)
    want = turned64(x, positions, freq)[0]
    y = rotary(x, None, positions, freq)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want)) and torch.isnan(y).sum() == 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("place", [lambda t: t, lambda t: torch.nn.functional.pad(t, (3, 5))[..., 3:-5]], ids=["contiguous", "off"])
def test_gradients(place, interleaved, dtype):
    freq, positions = rotary_frequencies(48, device=DEV)[0], torch.tensor([5, 0, 70000], device=DEV)
    q, k, dq, dk = (_randn(3, h, 64, dtype=dtype, seed=i) for i, h in enumerate((4, 2, 4, 2)))
    q, k = place(q).detach().requires_grad_(True), place(k).detach().requires_grad_(True)
    y, z = rotary(q, k, positions, freq, interleaved=interleaved, scale=1.5)
    gq, gk = torch.autograd.grad((y, z), (q, k), (place(dq), dk), retain_graph=True)
    _check(dq, gq, positions, freq, 1.5, interleaved, True)
    _check(dk, gk, positions, freq, 1.5, interleaved, True)
    # one output, one input, a broadcast gradient, nothing wanted
    assert torch.equal(torch.autograd.grad(y, q, dq, retain_graph=True)[0], gq) and torch.equal(torch.autograd.grad(z, k, dk, retain_graph=True)[0], gk)
    assert torch.autograd.grad(z, q, dk, allow_unused=True, retain_graph=True)[0] is None
    ones = torch.autograd.grad(y.sum() + z.sum(), (q, k))
    assert torch.equal(ones[1], torch.autograd.grad(rotary(k, None, positions, freq, interleaved=interleaved, scale=1.5), k, torch.ones_like(dk))[0])
    only = rotary(q.detach(), k, positions, freq, interleaved=interleaved, scale=1.5)
    assert torch.equal(torch.autograd.grad(only, k, (dq, dk), allow_unused=True)[0], gk)
    with torch.no_grad():
        assert not rotary(q, k, positions, freq)[0].requires_grad


@pytest.mark.parametrize("place", [lambda t: t, lambda t: torch.nn.functional.pad(t, (3, 5))[..., 3:-5]], ids=["contiguous", "off"])
def test_gradients_of_gradients_and_differences(place):
    """Turning is linear: differences are exact up to rounding, and the gradient of the gradient is the forward pass."""
    freq, positions = rotary_frequencies(32, device=DEV)[0], torch.tensor([3, 9], device=DEV)
    q = place(_randn(2, 2, 32, dtype=torch.float32)).detach().requires_grad_(True)
    y = rotary(q, None, positions, freq)
    dy = _randn(2, 2, 32, dtype=torch.float32, seed=1).requires_grad_(True)
    gq, = torch.autograd.grad(y, q, dy, create_graph=True)
    v = _randn(2, 2, 32, dtype=torch.float32, seed=2)
    again, = torch.autograd.grad(gq, dy, v)
    assert torch.equal(again, rotary(v, None, positions, freq))
    step = _randn(2, 2, 32, dtype=torch.float32, seed=3)
    with torch.no_grad():
        difference = (f64(rotary(q + step, None, positions, freq)) - f64(rotary(q - step, None, positions, freq))) / 2
    slope = (f64(gq) * f64(step)).sum()
    assert abs((difference * f64(dy)).sum() - slope) <= 128 * 2.0**-22 * ((f64(q).abs() + f64(step).abs()).max() * f64(dy).abs().max())


def test_hooks_on_saved_tensors_are_checked():
    freq, positions = rotary_frequencies(32, device=DEV)[0], torch.arange(4, device=DEV)
    for place in (lambda t: t, lambda t: torch.nn.functional.pad(t, (3, 5))[..., 3:-5]):
        q = place(_randn(4, 2, 32, dtype=torch.float32)).detach().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1]):
            y = rotary(q, None, positions, freq)
        with pytest.raises(RuntimeError, match="rotary: a saved tensor came back"):
            y.sum().backward()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
            y = rotary(q, None, positions, freq)
        assert torch.equal(torch.autograd.grad(y.sum(), q)[0], torch.autograd.grad(rotary(q, None, positions, freq).sum(), q)[0])


def test_refusals():
    q, freq, positions = _randn(4, 2, 32, dtype=torch.bfloat16), rotary_frequencies(32, device=DEV)[0], torch.arange(4, device=DEV)
    for args, text in (((q, q[:2], positions, freq), "k of shape"), ((q, q.half(), positions, freq), "k is"), ((q, None, positions[:3], freq), "positions of shape"),
                       ((q, None, positions.float(), freq), "not int64"), ((q, None, positions.cpu(), freq), "positions on"), ((q, None, positions, freq.half()), "inv_freq is"),
                       ((q[..., :16], None, positions, freq), "pairs"), ((q, None, positions, freq.cpu()), "inv_freq on"), ((q[0, 0], None, positions, freq), "heads, dim"),
                       ((q, None, positions, freq.clone().requires_grad_(True)), "no gradient")):
        with pytest.raises(ValueError, match=text):
            rotary(*args)
    with pytest.raises(_lib.MilesQuantError, match="dtype"):
        rotary(q.double(), None, positions, freq)
    with pytest.raises(_lib.MilesQuantError, match="1024"):
        rotary(torch.zeros(4, 1, 1032, device=DEV), None, positions, freq)


def test_gradients_that_are_broadcast_unused_or_added_up():
    q, k = (_randn(2, 19, n, 64, dtype=torch.bfloat16, seed=n).requires_grad_(True) for n in (4, 2))
    positions, freq = torch.arange(19, device=DEV) * 11, rotary_frequencies(64, device=DEV)[0]
    y, z = rotary(q, k, positions, freq)
    y.sum().backward()                                     # of ones that share one address; nothing for k
    assert k.grad is None and torch.equal(q.grad, rotary(torch.ones_like(q), None, positions, freq, inverse=True))
    y, z = rotary(q, q[:, :, :2], positions, freq)         # the same leaf as both
    dq = torch.autograd.grad((y.float().sum() + 2 * z.float().sum()), q)[0]
    ones = rotary(torch.ones_like(q), None, positions, freq, inverse=True).detach()
    assert torch.equal(dq[:, :, 2:], ones[:, :, 2:]) and torch.equal(dq[:, :, :2], 3 * ones[:, :, :2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
def test_results_that_go_past_the_caches(interleaved, dtype):
    q, k = (_randn(1, 4099, n, 128, dtype=dtype, seed=n) for n in (12, 4))
    positions, freq = torch.arange(4099, device=DEV) * 31, rotary_frequencies(96, device=DEV)[0]
    for x, y in zip((q, k), rotary(q, k, positions, freq, interleaved=interleaved)):
        _check(x, y, positions, freq, 1.0, interleaved)


def test_more_tokens_than_a_launch_has():
    tokens = 16 * (1 << 23) + 4321
    x = torch.arange(tokens * 8, dtype=torch.int32, device=DEV).bfloat16().view(tokens, 1, 8)
    positions, freq = torch.arange(tokens, dtype=torch.int32, device=DEV) % 4096, rotary_frequencies(8, device=DEV)[0]
    y = rotary(x, None, positions, freq, interleaved=True)
    for part in (slice(0, 3000), slice(tokens - 6000, None)):
        assert torch.equal(y[part], rotary(x[part], None, positions[part].clone(), freq, interleaved=True))
