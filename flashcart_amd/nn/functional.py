"""Node-wise functions in float32, bfloat16 and float16: embedding lookup, gated
feed-forward block, residual dropout.

They have no counterpart among the reference's kernels (it composes torch operations). Each is a registered operator
(``torch.ops.flashcart.*``) with an autograd formula, runs on the current stream and allocates through torch, so it can
be captured into a graph. There is no CPU path, and there are no forward-mode derivatives (an argument with a tangent is
refused). Values are formed in float32 and outputs rounded once to the tensors' type; what the feed-forward block rounds
between its products stands there. None has an autocast rule: under ``torch.autocast`` the arguments keep their types.
"""

from typing import Optional

import torch

from flashcart_amd.nn import _node_ops

__all__ = ["dropout_add", "embedding", "gated_feed_forward"]


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]``.

    Args:
        ids: int64 or int32, any shape. An index outside the table gives a row of NaN (a kernel cannot raise) and takes
            no part in the gradient.
        table: (rows, width).
        scale: factor of every row.
        padding_idx: row that gets no gradient; negative counts from the end.

    Returns:
        (*ids.shape, width) in the table's type. The table's gradient adds the rows of each index in float32, in an order
        that the sizes and indices fix: it is the same in every run.
    """
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"`ids` must be int64 or int32, got {ids.dtype}.")
    rows = table.shape[0] if table.dim() == 2 else 0
    padding = -1
    if padding_idx is not None:
        padding = padding_idx + rows if padding_idx < 0 else padding_idx
        if not 0 <= padding < rows:
            raise ValueError(f"padding_idx={padding_idx} is outside the table of {rows} rows.")
    return _node_ops.ops().embedding.default(ids, table, float(scale), padding)


def gated_feed_forward(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, act: str = "silu",
                       act_scale: float = 1.0, scale_in: float = 1.0, scale_out: float = 1.0) -> torch.Tensor:
    """``scale_out * (act_scale * act(gate) * up) @ w_out.T`` with ``[gate | up] = scale_in * x @ w_in.T``.

    Args:
        x: (..., width).
        w_in: (2 hidden, width), the gate's rows first.
        w_out: (width, hidden).
        act: "silu", "sigmoid" or "gelu" (erf form).
        act_scale, scale_in, scale_out: factors, as the rescaled activations and linear layers of this package have them.

    Sums are float32. For bfloat16 and float16 the hidden values ``act(gate) * up`` and, in the backward pass, the
    gradients of gate and up are rounded to that type, being operands of the matrix instructions. The activation and
    its derivative are formed from unrounded values and kept for the backward pass with 16 significant bits (float32:
    all). Outputs and gradients are 1.4 times as far from exact ones as one rounding to the type. (float16: hidden values
    above 65,504 become infinite.) float32 products keep float32 accuracy (operands below 2^-116 lose bits); the
    activation's exponential has a relative error of about 2^-24 (1 + |gate|), which shows where silu and sigmoid
    vanish. In training the block keeps the hidden values
    and the activation's factors: 8 bytes per hidden value (14 for float32). There are no second derivatives.
    """
    if act not in _node_ops.ACTIVATIONS:
        raise ValueError(f"act must be one of {sorted(_node_ops.ACTIVATIONS)}, got {act!r}.")
    save = torch.is_grad_enabled() and (x.requires_grad or w_in.requires_grad or w_out.requires_grad)
    return _node_ops.ops().gated_feed_forward.default(x, w_in, w_out, _node_ops.ACTIVATIONS[act], float(act_scale),
                                                      float(scale_in), float(scale_out), save)[0]


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, rng: torch.Tensor) -> torch.Tensor:
    """``residual + dropout(x, p)`` from a counter-based generator, without a stored mask.

    Element e is kept when word e % 4 of the Philox4x32-10 block of counter (e // 4, offset) and key ``seed`` is at least
    floor(p 2^32); the backward pass forms the mask again.

    Args:
        x: any shape.
        residual: same shape and type, or None.
        p: probability of dropping an element, in [0, 1].
        rng: int64 tensor (seed, offset) on x's device. The caller advances the offset from call to call (on the device
            where the call is captured into a graph): the same pair gives the same mask.
    """
    return _node_ops.ops().dropout_add.default(x, residual, float(p), rng)
