"""Node-wise functions in float32, bfloat16 and float16: embedding lookup, gated
feed-forward block, residual dropout, root-mean-square norm, dense layers (also with a weight for each group of rows), and
the norm and dense layers of 8-bit inference.

They have no counterpart among the reference's kernels (it composes torch operations). Each is a registered operator
(``torch.ops.flashcart.*``) with an autograd formula, runs on the current stream and allocates through torch, so it can
be captured into a graph. There is no CPU path, and there are no forward-mode derivatives (an argument with a tangent is
refused). Values are formed in float32 and outputs rounded once to the tensors' type; what the feed-forward block and the
dense layers round between their products stands there. None has an autocast rule: under ``torch.autocast`` the arguments keep their types.
"""

from typing import Optional, Tuple

import torch

from flashcart_amd.nn import _node_ops

__all__ = ["dense", "dropout_add", "embedding", "gated_feed_forward", "grouped_dense", "quantize_rows", "quantized_dense",
           "rms_norm_add", "rms_norm_add_quantized"]


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


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _activation(act: Optional[str]) -> int:
    if act is None:
        return _node_ops.NO_ACTIVATION
    if act not in _node_ops.ACTIVATIONS:
        raise ValueError(f"act must be None or one of {sorted(_node_ops.ACTIVATIONS)}, got {act!r}.")
    return _node_ops.ACTIVATIONS[act]


def rms_norm_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(weight * total / sqrt(mean(total^2) + eps), total)`` with ``total = x + residual``.

    Args:
        x: (..., width).
        residual: as x, or None: the total is x itself.
        weight: (width) of x's type, or None for ones.

    The norm is that of the total as it is returned, rounded to the tensors' type. Both outputs have gradients; the
    weight's adds its rows in float32 in an order that the sizes fix. There are no second derivatives. A row of zeros with
    ``eps=0`` gives NaN. Squares are summed in float32: a row whose sum leaves it gives zeros.
    """
    y, total, _ = _node_ops.ops().rms_norm_add.default(x, residual, weight, float(eps), _wants_grad(x, residual, weight))
    return y, x if residual is None else total


def rms_norm_add_quantized(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                           weight: Optional[torch.Tensor] = None,
                           eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``rms_norm_add`` with its norm in 8 bits, for inference: (q, scale, total), the norm being ``q * scale[..., None]``.

    scale (float32) is ``max(|y|, 2^-100) / 448`` over the row, y being the unrounded norm. q is float8_e4m3fn, the number
    nearest to ``448 y / max(|y|, 2^-100)`` (for 16-bit types exactly, ties going to the even number; for float32 up to
    the rounding of y). A row with an infinity has an infinite square sum: NaN at the infinity, a norm of zero elsewhere and the
    least scale; with an infinity in the weight the scale is infinite, finite values give zero and infinite ones NaN. There are no gradients: arguments that
    require them are refused where autograd records.
    """
    q, scale, total = _node_ops.ops().rms_norm_add_quantized.default(x, residual, weight, float(eps))
    return q, scale, x if residual is None else total


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of the rows of x (..., width), as ``rms_norm_add_quantized`` gives them for its norm: the operands of
    ``quantized_dense``. A weight is laid out so once. A row with an infinity has an infinite scale, zeros, and NaN at the
    infinity."""
    return _node_ops.ops().quantize_rows.default(x)


def dense(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
          act_scale: float = 1.0, scale: float = 1.0, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + act_scale * act(scale * x @ weight.T + bias)``.

    Args:
        x: (..., in).
        weight: (out, in).
        bias: (out) or None.
        act: "silu", "sigmoid", "gelu" (erf form) or None.
        act_scale, scale: factors, as the rescaled activations and linear layers of this package have them.
        residual: (..., out) or None.

    Sums are float32, and bias, activation and residual are applied before the one rounding of the output. For bfloat16
    and float16 the gradient of the activation's argument is rounded to that type in the backward pass, being an operand of
    the matrix instructions (gradients of x and weight are 1.4 times as far from exact ones as one rounding; in float16 it is zero
    below 2^-25, as any float16 gradient is: scale the loss); the
    activation's derivative is kept for it with 11 significant bits beside bfloat16 (fewer for a derivative below 2^-29, none
    below 2^-40), 16 beside float16, in 2 and 3 bytes an output (float32: all, in 4). float32 products
    keep float32 accuracy, as in ``gated_feed_forward``; so does the activation. There are no second derivatives.
    """
    return _node_ops.ops().node_dense.default(x, weight, bias, residual, None, _activation(act), float(act_scale),
                                              float(scale), _wants_grad(x, weight, bias))[0]


def grouped_dense(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  act: Optional[str] = None, act_scale: float = 1.0, scale: float = 1.0) -> torch.Tensor:
    """``act_scale * act(scale * x[r] @ weight[e].T + bias[e])`` for each row r of group e, as ``dense`` without a residual.

    Args:
        x: (rows, in), the rows of a group together.
        weight: (groups, out, in).
        offsets: (groups + 1) int64 or int32 on x's device: group e has the rows ``offsets[e]`` to ``offsets[e + 1] - 1``.
            They are not read on the host. Groups may be empty; rows in front of the first and behind the last give zeros
            and take no part in gradients. Offsets outside the rows are taken as the nearest inside, one smaller than those
            before it as the largest of them.
        bias: (groups, out) or None.

    Returns:
        (rows, out). The gradients of a group without rows are zero.
    """
    if offsets is None:
        raise TypeError("`offsets` must be a tensor.")
    return _node_ops.ops().node_dense.default(x, weight, bias, None, offsets, _activation(act), float(act_scale),
                                              float(scale), _wants_grad(x, weight, bias))[0]


def quantized_dense(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                    bias: Optional[torch.Tensor] = None, act: Optional[str] = None, act_scale: float = 1.0,
                    scale: float = 1.0, residual: Optional[torch.Tensor] = None,
                    dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dense`` in 8 bits, for inference: x (..., in) and weight (out, in) in float8_e4m3fn with a float32 scale for each
    row, (...) and (out), as ``rms_norm_add_quantized`` and ``quantize_rows`` give them.

    Bias, residual and output have the type ``dtype``, bfloat16 or float16. The 8-bit matrix instructions add eight products
    with 13 bits below the largest's leading bit and those sums in float32: about 1.5e-5 of the output, below its rounding.
    There are no gradients: arguments that require them are refused where autograd records.
    """
    return _node_ops.ops().quantized_dense.default(x, x_scale, weight, weight_scale, bias, residual, _activation(act),
                                                   float(act_scale), float(scale), dtype)
