"""The node-wise layers under activation checkpointing, on the kernels."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("reentrant", [True, False])
def test_checkpointed_network(reentrant):
    """Output and gradients are those of the plain call bit for bit where the random numbers are handed in; without them the
    second run is refused."""
    from flashcart_amd.nn import NodeNetwork
    torch.manual_seed(1)
    net = NodeNetwork(30, 48, 72, depth=2, p=0.3, seed=4).to(DEV)
    ids = torch.randint(0, 30, (5, 40), device=DEV)
    out = net(ids)
    want = torch.autograd.grad(out.square().sum(), list(net.parameters()))
    for layer in net.dropouts:
        layer.rng[1] = 0
    start = torch.zeros((), device=DEV, requires_grad=True)  # (the reentrant kind wants a differentiable argument)
    again = checkpoint(lambda s, i, r: net(i, r) + s, start, ids, net.draw(), use_reentrant=reentrant)
    assert torch.equal(again, out)
    again.square().sum().backward()
    for p, w in zip(net.parameters(), want):
        assert torch.equal(p.grad, w)
    assert all(layer.rng[1].item() == 1 for layer in net.dropouts)
    out = checkpoint(lambda s, i: net(i) + s, start, ids, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="during a backward pass"):
        out.sum().backward()
