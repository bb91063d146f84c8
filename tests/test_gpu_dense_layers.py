"""Layers of the row norm and the dense layers as programs hold them: batches without rows."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("per_element", [False, True])
@pytest.mark.parametrize("shape", [(0,), (0, 3), (2, 0)])
def test_network_without_rows(shape, per_element):
    from flashcart_amd.nn import NormNodeNetwork
    net = NormNodeNetwork(5, 16, 24, per_element=per_element).to(DEV)
    out = net(torch.zeros(shape, dtype=torch.int64, device=DEV))
    assert out.shape == (*shape, 16)
    grads = torch.autograd.grad(out, list(net.parameters()), torch.zeros_like(out))
    assert all(g.shape == p.shape and not g.any() for g, p in zip(grads, net.parameters()))


@pytest.mark.parametrize("shape", [(0,), (0, 3)])
def test_eight_bit_network_without_rows(shape):
    from flashcart_amd.nn import NormNodeNetwork, QuantizedNodeNetwork
    net = QuantizedNodeNetwork(NormNodeNetwork(5, 16, 24).to(DEV))
    assert net(torch.zeros(shape, dtype=torch.int64, device=DEV)).shape == (*shape, 16)
