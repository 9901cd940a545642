"""A layer's matrix product with its epilogue, forward and backward, on the tensor cores
(``rfm_linear_forward`` / ``rfm_linear_backward``).

``linear`` computes ``act(x W^T + bias) + residual`` in one pass over the output: the projections and
feed-forward products of the decoder's and encoder's layers.  bfloat16 and float16 operands, float32
sums and epilogue, one rounding at the store; the backward's weight and bias gradients are summed in a
fixed order (the same bits on every run).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._native import host, reaches_kernels

#: ``activation`` values.
ACTIVATIONS = _lib.ACTIVATIONS


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x W^T + bias) + residual``, differentiable (once) in all four.

    ``x`` ``[..., in]`` and ``weight`` ``[out, in]`` bfloat16 or float16 (under autocast they are cast to its
    type first); ``bias`` ``[out]`` of that type or float32; ``residual`` ``[..., out]`` of that type.
    ``activation`` is ``"none"``, ``"relu"`` or ``"gelu"`` (the exact one).  Any sizes and strides: operands
    whose rows are not 16-byte aligned (an odd number of columns) are copied into padded rows first.
    """
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return host().linear(x, weight, bias, code, residual)


_TYPES = {torch.bfloat16, torch.float16}
_LAYER_FORWARD = torch.nn.Linear.forward
_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _only_a_product(layer: torch.nn.Module) -> bool:
    """Whether calling ``layer`` is ``x W^T + b`` on its parameters and nothing else: no subclass, adapter,
    parametrisation or forward of its own, and no hooks."""
    return (type(layer) is torch.nn.Linear and torch.nn.Linear.forward is _LAYER_FORWARD
            and "forward" not in layer.__dict__ and layer._compiled_call_impl is None
            and not any(getattr(layer, k) for k in _HOOKS) and not torch.nn.modules.module._has_any_global_hook())


def project(layer: torch.nn.Module, x: torch.Tensor) -> torch.Tensor:
    """``layer(x)`` through ``linear`` where the layer is a plain ``torch.nn.Linear`` whose product runs in 16
    bits (under a 16-bit autocast, or on 16-bit tensors); any other call stays with the layer."""
    if not _only_a_product(layer) or not reaches_kernels(x, layer.weight, layer.bias):
        return layer(x)
    weight, bias = layer.weight, layer.bias
    if torch.is_autocast_enabled("cuda"):
        # autocast leaves float64 operands alone, and so the product stays in 64 bits
        lowered = {torch.float32, *_TYPES}
        kernels = (torch.get_autocast_dtype("cuda") in _TYPES
                   and all(t is None or t.dtype in lowered for t in (x, weight, bias)))
    else:
        kernels = (x.dtype in _TYPES and weight.dtype == x.dtype
                   and (bias is None or bias.dtype in (x.dtype, torch.float32)))
    return linear(x, weight, bias) if kernels else layer(x)


def check_faults(device: torch.device | int | None = None) -> None:
    """Raise if a product on ``device`` (the current one) ever gave up a bounded wait, which leaves its
    output incomplete.  Never expected, and reported here only: a program that wants to know asks, between
    steps.  Waits for all of the device's streams; the mark stays for the rest of the process."""
    faults = ctypes.c_int(0)
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        _lib.check("rfm_linear_faults", _lib.load().rfm_linear_faults(ctypes.byref(faults)))
    if faults.value:
        raise RuntimeError("a matrix product gave up a bounded wait: its output is incomplete")
