"""Network layers: radial basis/cutoff, interaction, product, gates, norms, readout; node-wise embedding, feed-forward
block and dropout (their functions: ``flashcart_amd.nn.functional``)."""

from flashcart_amd.nn.radial import BesselBasis, ChebyshevBasis, PolynomialCutoff
from flashcart_amd.nn.layers import (
    EnergyReadoutLayer,
    EquivariantGatedLayer,
    InteractionLayer,
    LinearLayer,
    ProductLayer,
    RescaledSiLULayer,
    RMSLayerNorm,
    ScaleShiftEnergyLayer,
)
from flashcart_amd.nn.node_layers import (
    EmbeddingLayer,
    GatedFeedForwardLayer,
    NodeNetwork,
    ResidualDropoutLayer,
)

__all__ = [
    "BesselBasis",
    "ChebyshevBasis",
    "PolynomialCutoff",
    "EnergyReadoutLayer",
    "EquivariantGatedLayer",
    "InteractionLayer",
    "LinearLayer",
    "ProductLayer",
    "RescaledSiLULayer",
    "RMSLayerNorm",
    "ScaleShiftEnergyLayer",
    "EmbeddingLayer",
    "GatedFeedForwardLayer",
    "NodeNetwork",
    "ResidualDropoutLayer",
]
