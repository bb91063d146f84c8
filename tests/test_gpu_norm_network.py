"""The row norm and the dense layers together: a network against its formula in float64, with weights for each element too,
trained in a captured graph, and in 8 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SILU = 1.6765324703310907


def _network(per_element, dtype=torch.float32, n=12, width=24, hidden=40):
    from flashcart_amd.nn import NormNodeNetwork
    torch.manual_seed(3)
    net = NormNodeNetwork(n, width, hidden, depth=2, per_element=per_element, padding_idx=0)
    with torch.no_grad():
        for name, p in net.named_parameters():
            if "norms" in name:
                p += 0.2 * torch.randn_like(p)
            elif "bias" in name:
                p.normal_()
    return net.to(DEV, dtype)


def _formula(net, ids):
    """Output and the leaves (float64, on the CPU) of the network's parameters."""
    leaves = {k: p.detach().double().cpu().requires_grad_(True) for k, p in net.named_parameters()}
    ids = ids.cpu()
    x = leaves["embedding.weight"][ids]

    def norm(t, k):
        return leaves[f"norms.{k}.weight"] * t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)

    for k in range(2):
        w, b, out = leaves[f"expand.{k}.weight"], leaves[f"expand.{k}.bias"], leaves[f"contract.{k}.weight"]
        y = norm(x, k)
        if w.dim() == 3:
            z = torch.einsum("...i,...oi->...o", y, w[ids]) * w.shape[-1] ** -0.5 + b[ids]
        else:
            z = y @ w.t() * w.shape[-1] ** -0.5 + b
        x = x + SILU * torch.nn.functional.silu(z) @ out.t() * out.shape[-1] ** -0.5
    return norm(x, 2), leaves


@pytest.mark.parametrize("per_element", [False, True])
def test_network_matches_its_formula(per_element):
    net = _network(per_element)
    ids = torch.randint(1, 12, (6, 31), device=DEV)
    out = net(ids)
    grad = torch.randn_like(out)
    got = dict(zip(dict(net.named_parameters()), torch.autograd.grad(out, list(net.parameters()), grad)))
    want, leaves = _formula(net, ids)
    assert out.shape == (6, 31, 24)
    assert float((out.double().cpu() - want).abs().max()) <= 1e-5 * float(want.abs().max())
    grads = dict(zip(leaves, torch.autograd.grad(want, list(leaves.values()), grad.double().cpu())))
    for name, g in grads.items():
        assert float((got[name].double().cpu() - g).norm()) <= 1e-5 * float(g.norm()), name


def test_elements_outside_the_layer_give_zeros():
    from flashcart_amd.nn import ElementDenseLayer, ElementRows
    torch.manual_seed(0)
    layer = ElementDenseLayer(3, 16, 8, "gelu", bias=True).to(DEV)
    ids = torch.tensor([2, -1, 0, 3, 2, 1, 7, 0], device=DEV)
    rows = ElementRows(ids, 3)
    x = torch.randn(8, 16, device=DEV, requires_grad=True)
    y = rows.unsort(layer(rows.sort(x), rows))
    inside = (ids >= 0) & (ids < 3)
    z = torch.bmm(x[inside][:, None], layer.weight[ids[inside]].transpose(1, 2))[:, 0] * 0.25 + layer.bias[ids[inside]]
    assert not y[~inside].any()
    assert torch.allclose(y[inside], torch.nn.functional.gelu(z), rtol=1e-5, atol=1e-6)
    (g,) = torch.autograd.grad(y.sum(), x)
    assert not g[~inside].any() and bool(g[inside].any(1).all())


@pytest.mark.parametrize("per_element", [False, True])
def test_training_in_a_graph(per_element):
    """Three replays of a captured training step as three eager ones, from the same start: the same weights, bit by bit."""
    ids = torch.randint(1, 12, (40, 9), device=DEV)
    target = torch.randn(40, 9, 24, device=DEV)
    ends = []
    for captured in (False, True):
        net = _network(per_element, torch.float32)
        opt = torch.optim.SGD(net.parameters(), lr=1e-3)

        def step():
            loss = (net(ids) - target).square().mean()
            opt.zero_grad(set_to_none=True)
            loss.backward()
            opt.step()

        if captured:
            start = [p.detach().clone() for p in net.parameters()]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
                opt.zero_grad(set_to_none=True)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
            with torch.no_grad():
                for p, s in zip(net.parameters(), start):
                    p.copy_(s)
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
        else:
            for _ in range(3):
                step()
        ends.append([p.detach().clone() for p in net.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*ends))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_network_in_eight_bits(dtype):
    """Each operand of a product is off by at most 2^-4 of a value of its row (uniform in that: 2^-4 / sqrt 3 in the mean of
    squares, less where the numbers' significands are large), which the products of independent errors keep: four products
    with two such operands, and the norms divide by a total whose first part is exact."""
    from flashcart_amd.nn import QuantizedNodeNetwork
    net = _network(False, n=30, width=256, hidden=512)
    small = QuantizedNodeNetwork(net, dtype)
    ids = torch.randint(1, 30, (8, 40), device=DEV)
    with torch.no_grad():
        want = net(ids).double()
    got = small(ids)
    assert got.dtype == dtype and got.shape == want.shape
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -4 / 3 ** 0.5 * 8 ** 0.5
    assert torch.equal(got, small(ids))


def test_eight_bits_refuse_weights_of_elements():
    from flashcart_amd.nn import QuantizedNodeNetwork
    with pytest.raises(ValueError, match="no form in 8 bits"):
        QuantizedNodeNetwork(_network(True))


def test_quantized_layer_takes_both_forms():
    """Rows in 8 bits with their scales, or rows that it quantizes itself: the same; without gradients."""
    from flashcart_amd.nn import DenseLayer, QuantizedDenseLayer
    torch.manual_seed(1)
    layer = DenseLayer(64, 48, "silu", bias=True).to(DEV, torch.bfloat16)
    small = QuantizedDenseLayer(layer)
    x = torch.randn(10, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    from flashcart_amd.nn import functional as F
    with pytest.raises(NotImplementedError, match="no derivatives"):
        small(x)
    with torch.no_grad():
        y = small(x, residual=torch.ones(10, 48, device=DEV, dtype=torch.bfloat16))
    assert torch.equal(y, small(*F.quantize_rows(x.detach()), residual=torch.ones(10, 48, device=DEV, dtype=torch.bfloat16)))
    far = (y - 1 - layer(x)).detach().double()
    assert float(far.norm() / layer(x).detach().double().norm()) <= 2.0 ** -4 / 3 ** 0.5 * 2
