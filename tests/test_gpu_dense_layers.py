"""Layers of the row norm and the dense layers as programs hold them: batches without rows, changes of type and device."""

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


@pytest.mark.parametrize("change", [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.float(),
                                    lambda m: m.cpu().half().to(DEV), lambda m: torch.nn.Sequential(m).half()[0]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_eight_bit_modules_keep_their_types(change, dtype):
    from flashcart_amd.nn import DenseLayer, NormNodeNetwork, QuantizedDenseLayer, QuantizedNodeNetwork
    torch.manual_seed(2)
    x = torch.randn(7, 16, device=DEV).to(dtype)
    layer = QuantizedDenseLayer(DenseLayer(16, 24, "silu", bias=True).to(DEV), dtype)
    net = QuantizedNodeNetwork(NormNodeNetwork(5, 16, 24).to(DEV), dtype)
    ids = torch.randint(0, 5, (9,), device=DEV)
    want = layer(x), net(ids)
    types = [[b.dtype for b in m.buffers()] for m in (layer, net)]
    layer, net = change(layer), change(net)
    assert types == [[b.dtype for b in m.buffers()] for m in (layer, net)]
    assert torch.equal(layer(x), want[0]) and torch.equal(net(ids), want[1])
