"""The node-wise layers on the CPU, their functions replaced by differentiable statements in torch: which random numbers
they use, where a call is run again too."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from flashcart_amd.nn import NodeNetwork, ResidualDropoutLayer, functional
from oracle import node_ops as O


@pytest.fixture
def drawn(monkeypatch):
    """Replaces the functions; gives the (seed, offset) pairs that dropout is called with."""
    calls = []

    def dropout_add(x, residual, p, rng):
        calls.append(tuple(rng.tolist()))
        keep = O.dropout_keep(x.numel(), p, *rng.tolist()).view(x.shape)
        return residual + torch.where(keep, x / (1 - p), 0.0)

    def feed_forward(x, w_in, w_out, act, c, s_in, s_out):
        gate, up = (s_in * x @ w_in.t()).chunk(2, -1)
        return s_out * (c * torch.nn.functional.silu(gate) * up) @ w_out.t()

    monkeypatch.setattr(functional, "dropout_add", dropout_add)
    monkeypatch.setattr(functional, "gated_feed_forward", feed_forward)
    monkeypatch.setattr(functional, "embedding", lambda ids, table, scale, padding: scale * table[ids])
    return calls


KINDS = [True, False]  # use_reentrant


@pytest.mark.parametrize("reentrant", KINDS)
def test_masks_of_a_checkpointed_layer(reentrant, drawn):
    """With the numbers handed in, the gradient is that of the mask of the forward pass; two calls under way at once."""
    layer = ResidualDropoutLayer(0.5, seed=3)
    x = [torch.randn(40, 8, requires_grad=True) for _ in range(2)]
    outs = [checkpoint(lambda t, rng: layer(t, torch.zeros_like(t), rng), t, layer.draw(), use_reentrant=reentrant)
            for t in x]
    assert drawn == [(3, 0), (3, 1)]
    for k, (t, out) in enumerate(zip(x, outs)):
        t.grad = None
        out.sum().backward()
        keep = O.dropout_keep(t.numel(), 0.5, 3, k).view(t.shape)
        assert torch.equal(out.detach(), torch.where(keep, 2 * t.detach(), 0.0))
        assert torch.equal(t.grad, 2.0 * keep)
    assert drawn == [(3, 0), (3, 1), (3, 0), (3, 1)]
    assert layer.rng.tolist() == [3, 2]


@pytest.mark.parametrize("reentrant", KINDS)
def test_a_second_run_without_its_numbers_is_refused(reentrant, drawn):
    layer = ResidualDropoutLayer(0.5)
    x = torch.randn(5, 8, requires_grad=True)
    out = checkpoint(lambda t: layer(t, torch.zeros_like(t)), x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="during a backward pass"):
        out.sum().backward()
    assert x.grad is None and layer.rng.tolist() == [0, 1]
    layer.eval()  # no numbers are drawn: nothing to refuse
    checkpoint(lambda t: layer(t, t), x, use_reentrant=reentrant).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))


@pytest.mark.parametrize("reentrant", KINDS)
def test_gradients_of_a_checkpointed_network(reentrant, drawn):
    torch.manual_seed(0)
    net = NodeNetwork(9, 12, 20, depth=2, p=0.25, seed=11)
    ids = torch.randint(0, 9, (6, 5))
    out = net(ids)
    want = torch.autograd.grad(out.square().sum(), list(net.parameters()))
    net.dropouts[0].rng[1] = net.dropouts[1].rng[1] = 0
    del drawn[:]
    rng = net.draw()
    assert rng.tolist() == [[11, 0], [12, 0]]
    start = torch.zeros((), requires_grad=True)  # (the reentrant kind wants a differentiable argument)
    again = checkpoint(lambda s, i, r: net(i, r) + s, start, ids, rng, use_reentrant=reentrant)
    assert torch.equal(again, out)
    net.zero_grad()
    again.square().sum().backward()
    assert drawn == [(11, 0), (12, 0)] * 2
    for p, w in zip(net.parameters(), want):
        assert torch.equal(p.grad, w)


def test_plain_calls_draw_as_before(drawn):
    """Every training call takes the next offset; evaluation takes none."""
    layer = ResidualDropoutLayer(0.5, seed=-2)
    x = torch.ones(4)
    layer(x, x), layer(x, x)
    layer.eval()
    assert torch.equal(layer(x, x), 2 * x)
    layer.train()
    layer(x, x)
    assert drawn == [(-2, 0), (-2, 1), (-2, 2)] and layer.rng.tolist() == [-2, 3]


@pytest.mark.parametrize("reentrant", KINDS)
def test_a_compiled_layer_refuses_too(reentrant, monkeypatch):
    """The refusal is the operator's, when it runs: a layer compiled on its own and called in a checkpointed function."""
    monkeypatch.setattr(functional, "dropout_add", lambda x, residual, p, rng: residual + x * rng[1])
    layer = ResidualDropoutLayer(0.5)
    call = torch.compile(layer, backend="aot_eager", fullgraph=True)
    x = torch.randn(5, 8, requires_grad=True)
    z = torch.zeros(5, 8)
    for k in range(3):
        assert torch.equal(call(x, z), k * x)
    out = checkpoint(lambda t: call(t, z), x, use_reentrant=reentrant)
    assert torch.equal(out, 3 * x)
    with pytest.raises(RuntimeError, match="during a backward pass"):
        out.sum().backward()
    out = checkpoint(lambda t, rng: call(t, z, rng), x, layer.draw(), use_reentrant=reentrant)
    out.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 4.0)) and layer.rng.tolist() == [0, 5]


def test_compilers_trace_the_layer_whole():
    """One graph, which advances the buffer (and ends in the operator's own error on the CPU)."""
    seen = []

    def backend(graph, inputs):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op == "call_function")
        return graph.forward

    with pytest.raises(RuntimeError, match="ROCm devices only"):
        torch.compile(ResidualDropoutLayer(0.5), backend=backend, fullgraph=True)(torch.ones(4), torch.ones(4))
    assert any("dropout_add" in t for t in seen)
