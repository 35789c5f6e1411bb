"""What the graph nodes of the norms and linear layers that are written in Python rest on (no GPU needed)."""

import pytest
import torch

from miles_amd.kernels._rows import gradients_once, one_run, unpacked


class _Times(torch.autograd.Function):
    """x * w + r, its gradients as a kernel makes them: without a graph of their own"""

    @staticmethod
    def forward(ctx, x, w, r):
        ctx.save_for_backward(x, w)
        return x * w + r

    @staticmethod
    @gradients_once("times")
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        assert not torch.is_grad_enabled()
        return dy * w, dy * x if ctx.needs_input_grad[1] else None, dy


@pytest.mark.parametrize("loss", [torch.sum, lambda y: y.square().sum()], ids=["constant", "dependent"])
def test_gradients_of_gradients_are_refused_and_not_left_out(loss):
    x, w, r = (torch.randn(3, 4, generator=torch.Generator().manual_seed(i), requires_grad=True) for i in range(3))
    plain = torch.autograd.grad(loss(_Times.apply(x, w, r)), (x, w, r))
    y = _Times.apply(x, w, r)
    gx, gw, gr = torch.autograd.grad(loss(y), (x, w, r), create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(plain, (gx, gw, gr)))
    assert gx.requires_grad and gw.requires_grad
    for g in (gx, gw):
        with pytest.raises(RuntimeError, match="times: gradients of gradients are not supported"):
            torch.autograd.grad(loss(y) + g.square().sum(), (x, w), retain_graph=True)
    # the residual's gradient is the incoming one, whose graph goes through y once
    if gr.requires_grad:
        assert torch.allclose(torch.autograd.grad(gr.sum(), r)[0], torch.full_like(r, 2))
    gx = torch.autograd.grad(loss(_Times.apply(x, w.detach(), r)), x, create_graph=True)[0]
    assert gx.requires_grad


def test_a_saved_tensor_that_came_back_as_another_is_refused():
    t = torch.zeros(4, 6, dtype=torch.bfloat16)
    device = torch.device("cpu")
    assert unpacked(None, (4, 6), t.dtype, device, "linear") is None and unpacked(t, (4, 6), t.dtype, device, "linear") is t
    for other in (t.float(), t[:3], t[0], t.view(2, 12), t.to("meta")):
        with pytest.raises(RuntimeError, match="linear: a saved tensor came back as"):
            unpacked(other, (4, 6), t.dtype, device, "linear")
    for other in (t.t().contiguous().t(), torch.zeros(25, dtype=t.dtype)[1:].view(4, 6)):
        run = one_run(other)
        assert run.is_contiguous() and run.data_ptr() % 16 == 0 and torch.equal(run, t)
