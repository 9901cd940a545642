"""Layer norm over the last dimension, forward and backward, on the device
(``rfm_layer_norm_forward`` / ``rfm_layer_norm_backward``).

The decoder's and encoder's layers normalise every token between their attention and feed-forward
blocks.  ``layer_norm`` is ``torch.nn.functional.layer_norm`` over the last dimension for float32,
bfloat16 and float16 inputs: float32 arithmetic, one rounding at the stores, and weight and bias
gradients summed in float32 in a fixed order (the same bits on every run).
"""

from __future__ import annotations

import torch

from ._native import host


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    ``x`` ``[..., D]`` float32, bfloat16 or float16, any leading shape and strides (rows whose elements
    are not adjacent are copied first); ``weight`` and ``bias`` ``[D]`` of ``x``'s type or float32, both of
    one type, either of them None.  Returns ``x``'s shape and type, contiguous, differentiable (once) in
    all three.
    """
    return host().layer_norm(x, weight, bias, eps)
