"""The graph nodes of the norms and linear layers, in native code and in Python, under everything that torch does with a graph."""

import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint as recomputed

from miles_amd import _lib
from miles_amd.kernels.linear import linear
from miles_amd.kernels.norm import layer_norm, rms_norm
from miles_amd.kernels.quant.act_checkpoint import checkpoint_activation

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Declines:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture(params=["native", "python"])
def host(request, monkeypatch):
    """Both host layers: what is ordinary makes its node in native code, anything else in Python."""
    if request.param == "python":
        for module in ("miles_amd.kernels.linear", "miles_amd.kernels.norm", "miles_amd.kernels.quant.act_checkpoint", "miles_amd.utils.mxfp8"):
            monkeypatch.setattr(f"{module}.native", _Declines())
    return request.param


def _leaves(*shapes, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(DEV).requires_grad_(True) for s in shapes]


# name -> (shapes of the leaves, the call)
CALLS = {
    "linear": (((24, 64), (96, 64)), lambda x, w: linear(x, w)),
    "linear_few": (((3, 64), (96, 64), (96,)), lambda x, w, b: linear(x, w, b, activation="gelu")),
    "linear_residual": (((24, 64), (96, 64), (96,), (24, 96)), lambda x, w, b, r: linear(x, w, b, activation="silu", residual=r)),
    "linear_kept": (((24, 64), (96, 64), (96,), (24, 96)), lambda x, w, b, r: linear(x, w, b, activation="gelu_tanh", residual=r, checkpoint=True)),
    "layer_norm": (((24, 64), (64,), (64,)), lambda x, w, b: layer_norm(x, w, b)),
    "layer_norm_bias": (((24, 64), (64,)), lambda x, b: layer_norm(x, None, b)),
    "layer_norm_kept": (((24, 64), (64,), (64,)), lambda x, w, b: layer_norm(x, w, b, checkpoint=True)),
    "rms_norm": (((24, 64), (64,)), lambda x, w: rms_norm(x, w)),
    "rms_norm_kept": (((24, 64), (64,)), lambda x, w: rms_norm(x, w, checkpoint=True, output_checkpoint=True)[0]),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("loss", [lambda y: y.float().sum(), lambda y: y.float().square().sum()], ids=["constant", "dependent"])
def test_gradients_of_gradients_are_refused_and_not_left_out(name, loss, host):
    """A gradient that came out as a constant would leave a penalty on it out of the result without a word."""
    shapes, call = CALLS[name]
    leaves = _leaves(*shapes)
    plain = torch.autograd.grad(loss(call(*leaves)), leaves)
    y = call(*leaves)
    grads = torch.autograd.grad(loss(y), leaves, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(plain, grads))
    for i, g in enumerate(grads):
        if i == 3:                                         # a residual's gradient is the incoming one
            continue
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="gradients of gradients are not supported"):
            torch.autograd.grad(loss(y) + g.float().square().sum(), leaves, retain_graph=True)
        with pytest.raises(RuntimeError, match="gradients of gradients are not supported"):
            torch.autograd.grad(g.float().sum(), leaves, retain_graph=True, allow_unused=True)


def _loss(y):
    return (y.float() * torch.linspace(-1, 1, y.numel(), device=DEV).view(y.shape)).sum()


def _elsewhere(t):
    """The same values in other places: the last two dimensions the other way round in memory, or off 16 bytes."""
    if t.dim() > 1:
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    run = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return run.copy_(t)


@pytest.mark.parametrize("name", CALLS)
def test_hooks_on_saved_tensors(name, host):
    """What a hook gives back is read as it lies, and refused where it is not what was saved: the kernels have its address alone."""
    shapes, call = CALLS[name]
    leaves = _leaves(*shapes)
    want = torch.autograd.grad(_loss(call(*leaves)), leaves)
    with torch.autograd.graph.save_on_cpu():
        y = call(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(_loss(y), leaves)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), _elsewhere):
        y = call(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(_loss(y), leaves)))
    count = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: count.append(1) or t.detach(), lambda t: t):
        call(*leaves)
    for which in range(len(count)):
        for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t.reshape(-1)[: t.numel() // 2], lambda t: t.unsqueeze(0)):
            packed = []

            def pack(t):
                packed.append(t.detach())
                return len(packed) - 1

            with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: change(packed[i]) if i == which else packed[i]):
                y = call(*leaves)
            assert len(packed) == len(count)
            with pytest.raises(RuntimeError, match="a saved tensor came back as|weight has the input's type"):
                torch.autograd.grad(_loss(y), leaves)


def test_what_the_library_refuses_is_its_own_error_in_both_host_layers(host):
    x, w = (torch.zeros(1, 1 << 22, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for wanted in (False, True):
        with pytest.raises(_lib.MilesQuantError, match="linear: tensor too large"):
            linear(x.requires_grad_(wanted), w)
    assert linear(x[:, :64], w[:, :64]).shape == (1, 1)


@pytest.mark.parametrize("name", CALLS)
def test_an_input_written_between_forward_and_backward_is_noticed(name, host):
    shapes, call = CALLS[name]
    for which in range(len(shapes)):
        leaves = _leaves(*shapes)
        want = torch.autograd.grad(_loss(call(*leaves)), leaves)
        y = call(*leaves)
        with torch.no_grad():
            leaves[which].mul_(2)
        # x in 8 bits, or its normalized values, are the layer's own; a bias and a residual are not needed
        if (which == 0 and name.endswith("_kept")) or (which == 1 and name == "layer_norm_bias") or which >= 2:
            assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(_loss(y), leaves)))
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(_loss(y), leaves)


def test_a_copy_written_between_forward_and_backward_is_noticed(host):
    x, w = _leaves((24, 64), (96, 64))
    for part in ("codes", "scales"):
        kept = checkpoint_activation(x)
        y = linear(x, w, checkpoint=kept)
        getattr(kept, part).view(torch.uint8).zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(_loss(y), w)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_in_the_backward_pass(name, reentrant, host):
    shapes, call = CALLS[name]
    leaves = _leaves(*shapes)
    want = torch.autograd.grad(_loss(call(*leaves)), leaves)
    _loss(recomputed(call, *leaves, use_reentrant=reentrant)).backward()
    assert all(torch.equal(p, t.grad) for p, t in zip(want, leaves))


def test_calls_and_backward_passes_of_several_threads(host):
    per_thread = [{name: _leaves(*shapes, seed=i) for name, (shapes, _call) in CALLS.items()} for i in range(4)]

    def everything(mine):
        out = []
        for name, (_shapes, call) in CALLS.items():
            y = call(*mine[name])
            out += [y.detach(), *torch.autograd.grad(_loss(y), mine[name])]
        return out

    want = [everything(mine) for mine in per_thread]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = everything(per_thread[i])
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                wrong.append(i)
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


class _Tagged(torch.Tensor):
    """A subclass: never taken by the native layer."""


@pytest.mark.parametrize("name", CALLS)
def test_transforms_are_refused_and_subclasses_are_not(name):
    shapes, call = CALLS[name]
    leaves = [t.detach() for t in _leaves(*shapes)]
    x, rest = leaves[0], leaves[1:]
    wanted = [t.clone().requires_grad_(True) for t in leaves]

    def batched_gradients(y):
        return torch.autograd.grad(y, wanted, torch.stack([y.detach(), y.detach()]), is_grads_batched=True)

    for transformed in (lambda: torch.func.grad(lambda a: call(a, *rest).float().sum())(x),
                        lambda: torch.func.grad(lambda a: call(x, a, *rest[1:]).float().sum())(rest[0]),
                        lambda: torch.func.vmap(lambda a: call(a, *rest))(torch.stack([x, x])),
                        lambda: torch.func.vmap(lambda a: call(x, a, *rest[1:]))(torch.stack([rest[0], rest[0]])),
                        lambda: torch.func.jvp(lambda a: call(a, *rest), (x,), (x,)),
                        lambda: batched_gradients(call(*wanted))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            transformed()
    tagged = call(x.as_subclass(_Tagged).requires_grad_(True), *rest)
    assert torch.equal(tagged.detach().as_subclass(torch.Tensor), call(*leaves))


@pytest.mark.parametrize("name", CALLS)
def test_compiled_functions_call_them_as_they_are(name):
    shapes, call = CALLS[name]
    leaves = _leaves(*shapes)
    torch._dynamo.reset()
    compiled = torch.compile(lambda *a: call(*a) * 2, backend="eager")
    y = compiled(*leaves)
    want = call(*leaves) * 2
    assert torch.equal(y, want)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(_loss(y), leaves), torch.autograd.grad(_loss(want), leaves)))


class _Drops(torch.autograd.Function):
    """Hands no gradient back."""

    @staticmethod
    def forward(ctx, y):
        return y.clone()

    @staticmethod
    def backward(ctx, g):
        return None


@pytest.mark.parametrize("name", CALLS)
def test_no_gradient_from_downstream_counts_as_zeros(name, host):
    shapes, call = CALLS[name]
    leaves = _leaves(*shapes)
    grads = torch.autograd.grad(_loss(_Drops.apply(call(*leaves))), leaves, allow_unused=True)
    assert all(g is None or (g == 0).all() for g in grads)


# sizes whose products are cut along k, whose rows end off 16 bytes or inside a tile, and that have more rows than sets of lanes
WIDE = {
    "linear_cut": (((48, 4096), (520, 4096), (520,), (48, 520)), lambda x, w, b, r: linear(x, w, b, activation="gelu", residual=r)),
    "linear_cut_kept": (((333, 2048), (96, 2048), (96,), (333, 96)), lambda x, w, b, r: linear(x, w, b, activation="silu", residual=r, checkpoint=True)),
    "linear_large": (((1100, 2112), (2080, 2112), (2080,), (1100, 2080)), lambda x, w, b, r: linear(x, w, b, activation="gelu", residual=r, checkpoint=True)),
    "linear_odd": (((301, 777), (131, 777), (131,), (301, 131)), lambda x, w, b, r: linear(x, w, b, activation="gelu", residual=r)),
    "norm_odd": (((2100, 1031), (1031,), (1031,)), lambda x, w, b: layer_norm(x, w, b)),
    "norm_kept": (((700, 2080), (2080,), (2080,)), lambda x, w, b: layer_norm(x, w, b, checkpoint=True)),
    "norm_long": (((5, 33001), (33001,), (33001,)), lambda x, w, b: layer_norm(x, w, b)),
}


@pytest.mark.parametrize("name", {**CALLS, **WIDE})
def test_scratch_memory_is_written_before_it_is_read(name, host):
    """Fresh memory filled with NaNs, as torch does on demand: nothing of it comes out."""
    shapes, call = {**CALLS, **WIDE}[name]
    leaves = _leaves(*shapes)
    y = call(*leaves)
    want = [y, *torch.autograd.grad(_loss(y), leaves)]
    torch.use_deterministic_algorithms(True)
    try:
        y = call(*leaves)
        got = [y, *torch.autograd.grad(_loss(y), leaves)]
    finally:
        torch.use_deterministic_algorithms(False)
    assert not any(t.isnan().any() for t in want) and all(torch.equal(p, q) for p, q in zip(got, want))
