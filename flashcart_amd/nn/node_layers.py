"""Layers over the node-wise functions: element/token embedding, gated feed-forward block, residual dropout, and a small
network of them. They have no counterpart in the reference; parameters follow its conventions (normal weights, scaled by
the inverse square root of the layer's inputs in the forward pass, rescaled activations)."""

from typing import Optional

import torch
import torch.nn as nn

from flashcart_amd.nn import _node_ops, functional
from flashcart_amd.nn.layers import SIGMOID_SCALE, SILU_SCALE

_ACT_SCALE = {"silu": SILU_SCALE, "sigmoid": SIGMOID_SCALE, "gelu": 1.0}


class EmbeddingLayer(nn.Module):
    """``scale * weight[ids]`` (``functional.embedding``); the row ``padding_idx`` starts at zero and is not trained."""

    def __init__(self, n_rows: int, width: int, scale: float = 1.0, padding_idx: Optional[int] = None):
        super().__init__()
        self.scale = float(scale)
        self.padding_idx = padding_idx
        self.weight = nn.Parameter(torch.randn(n_rows, width))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx] = 0.0

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return functional.embedding(ids, self.weight, self.scale, self.padding_idx)


class GatedFeedForwardLayer(nn.Module):
    """``functional.gated_feed_forward`` with weights ``w_in`` (2 hidden, width), the gate's rows first, and ``w_out``."""

    def __init__(self, width: int, hidden: int, activation: str = "silu"):
        super().__init__()
        if activation not in _ACT_SCALE:
            raise ValueError(f"activation must be one of {sorted(_ACT_SCALE)}. Provided: {activation}.")
        self.activation = activation
        self.scale_in, self.scale_out = float(width) ** -0.5, float(hidden) ** -0.5
        self.w_in = nn.Parameter(torch.randn(2 * hidden, width))
        self.w_out = nn.Parameter(torch.randn(width, hidden))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return functional.gated_feed_forward(x, self.w_in, self.w_out, self.activation, _ACT_SCALE[self.activation],
                                             self.scale_in, self.scale_out)


class ResidualDropoutLayer(nn.Module):
    """``residual + dropout(x)`` in training, ``residual + x`` in evaluation. The generator's seed and offset are a buffer on
    the device that every training call advances there, so a captured graph draws new masks at each replay and a
    checkpoint goes on where it stopped.

    Layers of equal seed and offset draw the same mask: layers of one network need different seeds, and so do the processes
    of data-parallel training (whose wrapper must not copy this buffer from one process to the others).

    A call that is run again during the backward pass (activation checkpointing) has to draw the mask of the first run,
    which the buffer no longer holds. Hand it to both: ``rng = layer.draw()`` before, ``layer(x, residual, rng)`` inside what
    is run again. ``draw``, and so a training call without ``rng``, is refused during a backward pass."""

    def __init__(self, p: float, seed: int = 0):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1]. Provided: {p}.")
        self.p = float(p)
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))

    def draw(self) -> torch.Tensor:
        """Seed and offset of one call; the next one gets the next offset."""
        return _node_ops.ops().dropout_draw.default(self.rng)

    def forward(self, x: torch.Tensor, residual: torch.Tensor, rng: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return residual + x
        return functional.dropout_add(x, residual, self.p, self.draw() if rng is None else rng)


class NodeNetwork(nn.Module):
    """Embedding, then ``depth`` blocks x + dropout(feed_forward(x)). The dropouts' seeds are ``seed`` .. ``seed + depth - 1``:
    networks that are not to share masks need seeds that far apart."""

    def __init__(self, n_rows: int, width: int, hidden: int, depth: int = 2, p: float = 0.0, activation: str = "silu",
                 padding_idx: Optional[int] = None, seed: int = 0):
        super().__init__()
        self.embedding = EmbeddingLayer(n_rows, width, padding_idx=padding_idx)
        self.blocks = nn.ModuleList(GatedFeedForwardLayer(width, hidden, activation) for _ in range(depth))
        self.dropouts = nn.ModuleList(ResidualDropoutLayer(p, seed + k) for k in range(depth))

    def draw(self) -> torch.Tensor:
        """Seeds and offsets (depth, 2) of one call, for calls under activation checkpointing (``ResidualDropoutLayer``)."""
        return torch.stack([dropout.draw() for dropout in self.dropouts])

    def forward(self, ids: torch.Tensor, rng: Optional[torch.Tensor] = None) -> torch.Tensor:
        x = self.embedding(ids)
        for k, (block, dropout) in enumerate(zip(self.blocks, self.dropouts)):
            x = dropout(block(x), x, None if rng is None else rng[k])
        return x
