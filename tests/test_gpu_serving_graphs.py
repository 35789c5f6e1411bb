"""Rotary positions, appending and attention inside graphs, transforms and compiled functions, and calls larger than a launch."""

import pytest
import torch

from miles_amd.kernels.paged_attention import paged_attention
from miles_amd.kernels.paged_cache import PagedCache, append_tokens
from miles_amd.kernels.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rotary_inputs(tokens=37):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(2, tokens, n, 64, generator=g).bfloat16().to(DEV) for n in (4, 2))
    return q, k, torch.arange(tokens, device=DEV) * 5, rotary_frequencies(64)[0]


def _cache(kept8=False):
    g = torch.Generator().manual_seed(2)
    cache = PagedCache.empty(12, 16, 2, 64, kept8=kept8)
    k, v = (torch.randn(192, 2, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    with torch.no_grad():
        append_tokens(cache, k, v, torch.arange(192, device=DEV))
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(2, 6)
    return cache, table, torch.tensor([90, 33], dtype=torch.int32, device=DEV), torch.randn(2, 8, 64, generator=g).bfloat16().to(DEV)


def test_captured_rotary_forward_and_backward():
    q, k, positions, inv_freq = _rotary_inputs()
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def run(q, k, dq, dk):
        q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        y = rotary(q, k, positions, inv_freq)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (q, k), (dq, dk)))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run(q, k, dq, dk)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(q, k, dq, dk)
    for i in range(4):
        for t in (q, k, dq, dk):
            t.copy_(torch.randn(t.shape, device=DEV).bfloat16())
        positions.add_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, run(q, k, dq, dk)):
            assert torch.equal(got, want)


def test_transforms_and_forward_derivatives_are_refused():
    q, k, positions, inv_freq = _rotary_inputs()
    cache, table, lengths, x = _cache()
    wanted = [q.clone().requires_grad_(True), k.clone().requires_grad_(True)]

    def batched_gradients(y):
        return torch.autograd.grad(y, wanted, [torch.stack([t.detach(), t.detach()]) for t in y], is_grads_batched=True)

    before = [t.clone() for t in (cache.keys, cache.values)]
    slots, new = torch.zeros(2, 1, dtype=torch.long, device=DEV), torch.randn(2, 1, 2, 64, device=DEV).bfloat16()
    for transformed in (lambda: torch.func.grad(lambda a: rotary(a, k, positions, inv_freq)[0].float().sum())(q),
                        lambda: torch.func.vmap(lambda a: rotary(a, None, positions, inv_freq))(torch.stack([q, q])),
                        lambda: torch.func.vmap(lambda a: rotary(q, a, positions, inv_freq))(torch.stack([k, k])),
                        lambda: torch.func.jvp(lambda a: rotary(a, None, positions, inv_freq), (q,), (q,)),
                        lambda: batched_gradients(rotary(*wanted, positions, inv_freq)),
                        lambda: torch.func.vmap(lambda a: paged_attention(a, cache, table, lengths))(torch.stack([x, x])),
                        lambda: torch.func.jvp(lambda a: paged_attention(a, cache, table, lengths), (x,), (x,)),
                        lambda: torch.func.grad(lambda a: paged_attention(a, cache, table, lengths).float().sum())(x),
                        lambda: torch.func.vmap(lambda a, b: append_tokens(cache, a, a, b) or a)(new, slots)):
        with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
            transformed()
    assert all(torch.equal(t, b) for t, b in zip((cache.keys, cache.values), before))


def test_compiled_functions_call_them_as_they_are():
    q, k, positions, inv_freq = _rotary_inputs()
    torch._dynamo.reset()
    leaves = [q.requires_grad_(True), k.requires_grad_(True)]

    def turned(a, b):
        y, z = rotary(a, b, positions, inv_freq)
        return y * 2, z * 2

    made, want = torch.compile(turned, backend="eager")(*leaves), turned(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(made, want))
    grads = [torch.autograd.grad([t.float().square().sum() for t in y], leaves) for y in (made, want)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    for kept8 in (False, True):
        cache, table, lengths, x = _cache(kept8)
        new, slots = torch.randn(2, 2, 64, device=DEV).bfloat16(), torch.tensor([89, 96 + 32], device=DEV)

        def step(x, new, slots):
            append_tokens(cache, new, new, slots)
            return paged_attention(x, cache, table, lengths) * 2

        with torch.no_grad():
            assert torch.equal(torch.compile(step, backend="eager")(x, new, slots), step(x, new, slots))


@pytest.mark.parametrize("strided", [False, True], ids=["native", "python"])
def test_a_graph_that_saved_a_cache_notices_what_is_appended(strided):
    cache, _, _, _ = _cache()
    w = torch.ones((), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = (w * cache.values).sum()
    k, slots = torch.randn(4, 2, 64, device=DEV).bfloat16(), torch.arange(8, device=DEV)
    append_tokens(cache, k, k, slots[::2] if strided else slots[:4])
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    with torch.inference_mode():                          # whose tensors have no such count
        other = PagedCache.empty(4, 16, 2, 64)
        append_tokens(other, k, k, slots[:4].clone())
    append_tokens(other, k, k, slots[4:].clone())
    assert torch.equal(other.gather(torch.arange(8, device=DEV))[0], torch.cat([k, k]))


def test_more_heads_than_a_launch_has_lanes_for():
    """One token each for most of five million sequences, none for the others: a weight of one, so the value itself."""
    batch, heads = 5_000_000, 16
    cache = PagedCache.empty(3, 16, 1, 8)
    for t in (cache.keys, cache.values):
        t.copy_(torch.randn(t.shape, device=DEV))
    q = torch.randn(1, 1, 8, device=DEV).bfloat16().expand(batch, heads, 8)
    table = (torch.arange(batch, device=DEV) % 3).int().view(batch, 1)
    lengths = (torch.arange(batch, device=DEV) % 5 != 0).int()
    out = paged_attention(q, cache, table, lengths)
    want = cache.values[:, 0, 0][table[:, 0].long()] * lengths[:, None]
    assert all(torch.equal(out[:, h], want) for h in range(heads))
