"""The serving operators together, as a decoding program uses them: prompts appended, then tokens one by one, eagerly and out of a captured graph."""

import pytest
import torch

from miles_amd.kernels.linear import linear
from miles_amd.kernels.norm import rms_norm
from miles_amd.kernels.paged_attention import paged_attention
from miles_amd.kernels.paged_cache import PagedCache, append_tokens
from miles_amd.kernels.rotary import rotary, rotary_frequencies
from tests.operator_checks import within
from tests.serving_checks import DEV, attend64

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, HIDDEN, PAGE = 8, 2, 64, 256, 16


class _Layer:
    """norm, fused projection, rotation and append, attention, projection back onto the residual stream"""

    def __init__(self, kept8, seed=0):
        g = torch.Generator().manual_seed(seed)
        make = lambda *s: (torch.randn(s, generator=g) / s[-1] ** 0.5).bfloat16().to(DEV)  # noqa: E731
        self.gamma, self.qkv, self.out = torch.ones(HIDDEN, dtype=torch.bfloat16, device=DEV), make((HEADS + 2 * KV) * DIM, HIDDEN), make(HIDDEN, HEADS * DIM)
        self.freq = rotary_frequencies(DIM, device=DEV)[0]
        self.cache = PagedCache.empty(64, PAGE, KV, DIM, kept8=kept8, device=DEV)
        for t in (self.cache.keys, self.cache.values):
            t.copy_(torch.full(t.shape, float("nan")))

    def project(self, x):
        q, k, v = linear(rms_norm(x, self.gamma), self.qkv).split((HEADS * DIM, KV * DIM, KV * DIM), 1)
        return q.unflatten(1, (HEADS, DIM)), k.unflatten(1, (KV, DIM)), v.unflatten(1, (KV, DIM))

    def step(self, x, positions, slots, pages, lengths):
        q, k, v = self.project(x)
        q = append_tokens(self.cache, k, v, slots, positions=positions, inv_freq=self.freq, q=q)
        a = paged_attention(q, self.cache, pages, lengths)
        return linear(a.flatten(1), self.out, residual=x), q, a


@torch.no_grad()
@pytest.mark.parametrize("kept8", [False, True], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("width", [8, 64], ids=["whole", "shared"])
def test_prompts_and_then_tokens_one_by_one(width, kept8):
    layer, prompts = _Layer(kept8), [5, 0, 33, 16]
    batch = len(prompts)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    table[:, :8] = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:batch * 8].view(batch, 8).int().to(DEV)
    slot = lambda i, t: (table[i, t // PAGE].long() * PAGE + t % PAGE)  # noqa: E731
    history = [[] for _ in prompts]                        # of every sequence: keys (turned) and values of its tokens

    def note(i, k, v, at):
        history[i].append((rotary(k.float(), None, at, layer.freq), v))

    g = torch.Generator().manual_seed(2)
    for i, n in enumerate(prompts):
        at = torch.arange(n, device=DEV)
        _, k, v = layer.project(torch.randn(n, HIDDEN, generator=g).bfloat16().to(DEV))
        append_tokens(layer.cache, k, v, slot(i, at), positions=at, inv_freq=layer.freq)
        note(i, k, v, at)
    # the fourth place of the batch is idle from the third step on: its slot is none, its length 0
    state = dict(x=torch.zeros(batch, HIDDEN, dtype=torch.bfloat16, device=DEV), positions=torch.zeros(batch, dtype=torch.int64, device=DEV),
                 slots=torch.full((batch,), -1, dtype=torch.int64, device=DEV), pages=table.clone(), lengths=torch.zeros(batch, dtype=torch.int32, device=DEV))
    graph, captured = torch.cuda.CUDAGraph(), None
    for step in range(40):
        lengths = [0 if i == 3 and step >= 3 else n + step + 1 for i, n in enumerate(prompts)]
        at = torch.tensor([max(0, n - 1) for n in lengths], device=DEV)
        state["x"].copy_(torch.randn(batch, HIDDEN, generator=g))
        state["positions"].copy_(at)
        state["slots"].copy_(torch.where(torch.tensor(lengths, device=DEV) > 0, torch.stack([slot(i, a) for i, a in enumerate(at)]), -1))
        state["lengths"].copy_(torch.tensor(lengths))
        if step == 2:                                      # captured with the lengths of this step, replayed with all later ones
            layer.step(**state)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                captured = layer.step(**state)
        before = [t.clone() for t in (layer.cache.keys, layer.cache.values)]
        if captured is not None:
            graph.replay()
            y, q, a = (t.clone() for t in captured)
            for now, old in zip((layer.cache.keys, layer.cache.values), before):
                now.copy_(old)
        y2, q2, a2 = layer.step(**state)
        if captured is not None:
            assert torch.equal(y, y2) and torch.equal(q, q2) and torch.equal(a, a2)
        _, k, v = layer.project(state["x"])
        for i, n in enumerate(lengths):
            if n == 0:
                assert (a2[i] == 0).all() and torch.equal(y2[i], state["x"][i])
                continue
            note(i, k[i:i + 1], v[i:i + 1], at[i:i + 1])
            if step % 13 == 0 or step == 39:
                past = torch.cat([h[0] for h in history[i]]), torch.cat([h[1] for h in history[i]])
                got = layer.cache.gather(slot(i, torch.arange(n, device=DEV)))
                if kept8:                                  # half a step of e4m3, at least of the group's smallest
                    for t, p in zip(got, past):
                        scale = p.float().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2) / 224
                        assert ((t.float() - p.float()).abs() <= p.float().abs() * 2.0**-4 + scale * 2.0**-10).all()
                else:
                    assert torch.equal(got[0], past[0].bfloat16()) and torch.equal(got[1], past[1])
                want, off = attend64(q2[i], *got)
                within(a2[i], want, off, f"step {step}, sequence {i}")


@torch.no_grad()
def test_two_graphs_two_streams_and_another_stream_than_the_tensors_own():
    """Workspaces belong to the call: graphs that run one behind the other and calls that run beside each other do not share them."""
    g = torch.Generator().manual_seed(0)
    cache = PagedCache.empty(400, 16, 2, 64, device=DEV)
    for t in (cache.keys, cache.values):
        t.copy_(torch.randn(t.shape, generator=g))
    table = torch.randperm(400, generator=g).int().view(2, 200).to(DEV)
    lengths = torch.tensor([3100, 700], dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, 8, 64, generator=g).bfloat16().to(DEV) for _ in range(2)]
    want = [paged_attention(q, cache, table, lengths) for q in qs]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in qs], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            outs.append(paged_attention(q, cache, table, lengths))
    for _ in range(3):
        for o in outs:
            o.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    beside = [[] for _ in qs]
    for _ in range(20):
        for s, q, b in zip(streams, qs, beside):
            with torch.cuda.stream(s):
                b.append(paged_attention(q, cache, table, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for b, w in zip(beside, want) for o in b)


@torch.no_grad()
def test_calls_inside_a_block_of_deferred_jobs_run_at_once():
    from miles_amd import launch

    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    freq, positions = rotary_frequencies(64, device=DEV)[0], torch.arange(3, device=DEV)
    cache = PagedCache.empty(2, 16, 4, 64, device=DEV)
    pages, lengths = torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)

    def calls():
        return [rotary(q, None, positions, freq), append_tokens(cache, q, q, positions, positions=positions, inv_freq=freq, q=q), paged_attention(q, cache, pages, lengths)]

    want = calls()
    with launch.deferred():
        got = calls()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
