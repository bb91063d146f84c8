"""Fit the energy of random alloys from their composition with the node-wise operators: the element embedding, gated
feed-forward blocks and residual dropout of ``flashcart_amd.nn.NodeNetwork``, summed over the atoms of each structure.

    python examples/node_network.py [--steps 200] [--dtype bfloat16]

Each structure holds up to 64 atoms of the elements 1 .. 8; index 0 pads. Its energy is a sum of atomic energies. The
training step (forward, backward, update) is captured into a graph once and replayed; the dropout masks differ from
replay to replay, because the generator's offset is advanced on the device.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from flashcart_amd.nn import LinearLayer, NodeNetwork  # noqa: E402


class CompositionEnergy(torch.nn.Module):
    def __init__(self, n_elements=9, width=64, hidden=128, p=0.1):
        super().__init__()
        self.network = NodeNetwork(n_elements, width, hidden, depth=2, p=p, padding_idx=0, seed=7)
        self.readout = LinearLayer(width, 1)

    def forward(self, ids):
        atoms = self.network(ids)  # (structures, atoms, width)
        energy = self.readout(atoms.reshape(-1, atoms.shape[-1]).float()).view(ids.shape)
        return (energy * (ids > 0)).sum(-1)


def main(steps=200, dtype=torch.float32, structures=512, atoms=64, lr=1e-2, log=print):
    """Mean absolute error per atom of the energy (in evaluation, without dropout) before and after training."""
    torch.manual_seed(0)
    device = "cuda"
    ids = torch.randint(0, 9, (structures, atoms), device=device)
    atomic = torch.randn(9, device=device)
    target = (atomic[ids] * (ids > 0)).sum(-1)
    model = CompositionEnergy().to(device)
    for module in (model.network.embedding, model.network.blocks):
        module.to(dtype)
    opt = torch.optim.Adam(model.parameters(), lr=lr, capturable=True)

    def step():
        loss = (model(ids) - target).square().mean() / atoms
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()

    def error():
        model.eval()
        with torch.no_grad():
            off = (model(ids) - target).abs().mean() / atoms
        model.train()
        return float(off)

    before = error()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
        opt.zero_grad(set_to_none=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(steps):
        graph.replay()
        if (k + 1) % 50 == 0:
            log(f"step {k + 1}: error {error():.4f} per atom")
    return before, error()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--dtype", choices=["float32", "bfloat16", "float16"], default="float32")
    args = parser.parse_args()
    first, last = main(args.steps, getattr(torch, args.dtype))
    print(f"mean absolute error per atom: {first:.4f} before, {last:.4f} after {args.steps} steps")
