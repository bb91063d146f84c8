"""Layers over the node-wise functions: element/token embedding, gated feed-forward block, residual dropout, row norm, dense
layers (with weights for each element too, and in 8 bits), and small networks of them. They have no counterpart in the reference; parameters follow its conventions (normal weights, scaled by
the inverse square root of the layer's inputs in the forward pass, rescaled activations)."""

from typing import Optional, Tuple

import torch
import torch.nn as nn

from flashcart_amd.nn import _node_ops, functional
from flashcart_amd.nn.layers import SIGMOID_SCALE, SILU_SCALE

_ACT_SCALE = {"silu": SILU_SCALE, "sigmoid": SIGMOID_SCALE, "gelu": 1.0}


def _act_scale(activation: Optional[str]) -> float:
    if activation is None:
        return 1.0
    if activation not in _ACT_SCALE:
        raise ValueError(f"activation must be None or one of {sorted(_ACT_SCALE)}. Provided: {activation}.")
    return _ACT_SCALE[activation]


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


class RowNormLayer(nn.Module):
    """``functional.rms_norm_add`` with a weight that starts at one: the norm of x + residual, and that total."""

    def __init__(self, width: int, eps: float = 1e-6):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(width))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        return functional.rms_norm_add(x, residual, self.weight, self.eps)

    def quantized(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """``functional.rms_norm_add_quantized`` with this weight, which takes no part in gradients here."""
        return functional.rms_norm_add_quantized(x, residual, self.weight.detach(), self.eps)


class DenseLayer(nn.Module):
    """``functional.dense``: residual + rescaled activation of x W^T in_features^-1/2 + bias, in the parameters' type."""

    def __init__(self, in_features: int, out_features: int, activation: Optional[str] = None, bias: bool = False):
        super().__init__()
        self.activation, self.act_scale, self.scale = activation, _act_scale(activation), float(in_features) ** -0.5
        self.weight = nn.Parameter(torch.randn(out_features, in_features))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return functional.dense(x, self.weight, self.bias, self.activation, self.act_scale, self.scale, residual)


class _FixedTypes(nn.Module):
    """A module whose buffers keep their types: ``.half()``, ``.to(dtype)`` and the like, also of a module that holds it, move it
    between devices alone."""

    def _apply(self, fn, recurse=True):
        kept = dict(self.named_buffers(recurse=False))
        super()._apply(fn, recurse)
        for name, before in kept.items():
            after = getattr(self, name)
            if after.dtype != before.dtype:
                setattr(self, name, before.to(after.device))
        return self


class QuantizedDenseLayer(_FixedTypes):
    """A ``DenseLayer`` on the GPU in 8 bits, for inference (``functional.quantized_dense``): its weight as float8_e4m3fn with a
    scale for each row, laid out here once, bias and output in ``dtype``. Arguments that ask for gradients are refused. The types
    stay as they are laid out here under ``.half()``, ``.to(dtype)`` and the like."""

    def __init__(self, layer: DenseLayer, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.activation, self.act_scale, self.scale, self.dtype = layer.activation, layer.act_scale, layer.scale, dtype
        weight, weight_scale = functional.quantize_rows(layer.weight.detach())
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", None if layer.bias is None else layer.bias.detach().to(dtype))

    def forward(self, x: torch.Tensor, x_scale: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x in 8 bits with its scales, or without ``x_scale`` in a type that is quantized here."""
        if x_scale is None:
            x, x_scale = functional.quantize_rows(x)
        return functional.quantized_dense(x, x_scale, self.weight, self.weight_scale, self.bias, self.activation,
                                          self.act_scale, self.scale, residual, self.dtype)


class _Permute(torch.autograd.Function):
    """Rows in another order; the gradient's rows go back without a sum."""

    @staticmethod
    def forward(ctx, x, order, inverse):
        ctx.save_for_backward(order, inverse)
        return x.index_select(0, order)

    @staticmethod
    def backward(ctx, grad):
        order, inverse = ctx.saved_tensors
        return _Permute.apply(grad, inverse, order), None, None


class ElementRows:
    """The order of rows by element, formed once for the ``ids`` (any shape) of a structure or batch: what the layers with
    weights for each element take. Rows whose id is outside 0 .. n_elements - 1 are in no group: those layers give zeros there."""

    def __init__(self, ids: torch.Tensor, n_elements: int):
        by_element, self.order = torch.sort(ids.reshape(-1), stable=True)
        self.inverse = torch.empty_like(self.order)
        self.inverse[self.order] = torch.arange(self.order.numel(), device=ids.device)
        self.offsets = torch.searchsorted(by_element, torch.arange(n_elements + 1, device=ids.device, dtype=by_element.dtype))

    def sort(self, x: torch.Tensor) -> torch.Tensor:
        """(..., width) as (rows, width) in the order of the elements."""
        return _Permute.apply(x.reshape(-1, x.shape[-1]), self.order, self.inverse)

    def unsort(self, x: torch.Tensor) -> torch.Tensor:
        """The rows of ``sort`` where they were."""
        return _Permute.apply(x, self.inverse, self.order)


class ElementDenseLayer(nn.Module):
    """``functional.grouped_dense``: a dense layer with a weight (and bias) for each element, on rows in ``ElementRows``'
    order."""

    def __init__(self, n_elements: int, in_features: int, out_features: int, activation: Optional[str] = None,
                 bias: bool = False):
        super().__init__()
        self.activation, self.act_scale, self.scale = activation, _act_scale(activation), float(in_features) ** -0.5
        self.weight = nn.Parameter(torch.randn(n_elements, out_features, in_features))
        if bias:
            self.bias = nn.Parameter(torch.zeros(n_elements, out_features))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, rows: ElementRows) -> torch.Tensor:
        return functional.grouped_dense(x, self.weight, rows.offsets, self.bias, self.activation, self.act_scale, self.scale)


class NormNodeNetwork(nn.Module):
    """Embedding, then ``depth`` blocks x + contract(expand(norm(x))) of dense layers, and a last norm. With ``per_element`` the
    expanding layers have weights for each element; the rows are sorted by element once, at the embedding. Each residual is added in
    the norm that follows."""

    def __init__(self, n_elements: int, width: int, hidden: int, depth: int = 2, activation: str = "silu",
                 per_element: bool = False, padding_idx: Optional[int] = None):
        super().__init__()
        self.n_elements, self.per_element = n_elements, per_element
        self.embedding = EmbeddingLayer(n_elements, width, padding_idx=padding_idx)
        self.norms = nn.ModuleList(RowNormLayer(width) for _ in range(depth + 1))
        self.expand = nn.ModuleList(
            ElementDenseLayer(n_elements, width, hidden, activation, bias=True) if per_element
            else DenseLayer(width, hidden, activation, bias=True) for _ in range(depth))
        self.contract = nn.ModuleList(DenseLayer(hidden, width) for _ in range(depth))

    def forward(self, ids: torch.Tensor, rows: Optional[ElementRows] = None) -> torch.Tensor:
        """(*ids.shape, width). ``rows``: the order of these ids, where the caller has formed it already."""
        if self.per_element:
            rows = ElementRows(ids, self.n_elements) if rows is None else rows
            x = rows.sort(self.embedding(ids))
        else:
            x = self.embedding(ids)
        y, total = self.norms[0](x)
        for norm, expand, contract in zip(self.norms[1:], self.expand, self.contract):
            hidden = expand(y, rows) if self.per_element else expand(y)
            y, total = norm(contract(hidden), total)
        return rows.unsort(y).view(*ids.shape, y.shape[-1]) if self.per_element else y


class QuantizedNodeNetwork(_FixedTypes):
    """A ``NormNodeNetwork`` on the GPU (not ``per_element``) for inference in 8 bits: the norms write what the expanding layers
    read, activations are quantized row by row between the layers, sums of blocks are in ``dtype``. The types stay so under
    ``.half()``, ``.to(dtype)`` and the like."""

    def __init__(self, network: NormNodeNetwork, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if network.per_element:
            raise ValueError("layers with weights for each element have no form in 8 bits.")
        self.dtype = dtype
        self.scale = network.embedding.scale
        self.register_buffer("table", network.embedding.weight.detach().to(dtype))
        for k, norm in enumerate(network.norms):
            self.register_buffer(f"norm{k}", norm.weight.detach().to(dtype))
        self.eps = [norm.eps for norm in network.norms]
        self.expand = nn.ModuleList(QuantizedDenseLayer(layer, dtype) for layer in network.expand)
        self.contract = nn.ModuleList(QuantizedDenseLayer(layer, dtype) for layer in network.contract)

    @torch.no_grad()
    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        delta, total = functional.embedding(ids, self.table, self.scale), None
        for k, (expand, contract) in enumerate(zip(self.expand, self.contract)):
            q, scale, total = functional.rms_norm_add_quantized(delta, total, getattr(self, f"norm{k}"), self.eps[k])
            delta = contract(expand(q, scale))
        last = len(self.expand)
        return functional.rms_norm_add(delta, total, getattr(self, f"norm{last}"), self.eps[last])[0]
