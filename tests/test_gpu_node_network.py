"""The node-wise layers together: a network against the float64 statement, and the example's training in a graph."""

import importlib.util
import os

import pytest
import torch

from oracle import node_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_network_matches_its_formula():
    """Output and parameter gradients of embedding and two blocks with dropout, float32 against autograd over the oracle's
    formulas in float64; then evaluation, and the masks of a second training call."""
    from flashcart_amd.nn import NodeNetwork
    torch.manual_seed(3)
    net = NodeNetwork(12, 24, 40, depth=2, p=0.25, padding_idx=0, seed=5).to(DEV)
    ids = torch.randint(0, 12, (6, 31), device=DEV)
    out = net(ids)
    grad = torch.randn_like(out)
    got = torch.autograd.grad(out, list(net.parameters()), grad)

    def formula(keeps):
        leaves = [p.detach().double().cpu().requires_grad_(True) for p in net.parameters()]
        table, (in0, out0, in1, out1) = leaves[0], leaves[1:]
        x = table[ids.cpu()]
        for (w_in, w_out), keep in zip(((in0, out0), (in1, out1)), keeps):
            gate, up = ((x @ w_in.t()) * 24 ** -0.5).chunk(2, -1)
            h = 1.6765324703310907 * torch.nn.functional.silu(gate) * up
            x = x + keep * ((h @ w_out.t()) * 40 ** -0.5)
        return x, leaves

    n = out.numel()
    keeps = [O.dropout_keep(n, 0.25, 5 + k, 0).view(out.shape) / 0.75 for k in range(2)]
    want, leaves = formula(keeps)
    assert float((out.double().cpu() - want).abs().max()) <= 1e-5 * float(want.abs().max())
    grads = torch.autograd.grad(want, leaves, grad.double().cpu())
    for g, w in zip(got, grads):
        w = w.clone()
        if w.shape == (12, 24):
            w[0] = 0  # the padding row is not trained
        assert float((g.double().cpu() - w).abs().max()) <= 1e-5 * float(w.abs().max())
    second = net(ids)
    keeps = [O.dropout_keep(n, 0.25, 5 + k, 1).view(out.shape) / 0.75 for k in range(2)]
    assert float((second.double().cpu() - formula(keeps)[0]).abs().max()) <= 1e-5 * float(want.abs().max())
    net.eval()
    plain = formula([torch.ones(())] * 2)[0]
    assert float((net(ids).double().cpu() - plain).abs().max()) <= 1e-5 * float(plain.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_trains(dtype):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "node_network.py")
    spec = importlib.util.spec_from_file_location("node_network", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    before, after = module.main(steps=150, dtype=dtype, log=lambda text: print(text, flush=True))
    assert after < 0.2 * before
