"""Layer norm over the last dimension, forward and backward, on the device
(``rfm_layer_norm_forward`` / ``rfm_layer_norm_backward``).

The decoder's and encoder's layers normalise every token between their attention and feed-forward
blocks.  ``layer_norm`` is ``torch.nn.functional.layer_norm`` over the last dimension for float32,
bfloat16 and float16 inputs: float32 arithmetic, one rounding at the stores, and weight and bias
gradients summed in float32 in a fixed order (the same bits on every run).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._launch import DTYPES, on_device, raw_stream, require_cuda, row_stride, rows_of


def _param_code(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None) -> int:
    p = weight if weight is not None else bias
    return DTYPES[x.dtype if p is None else p.dtype]


def _forward(x, weight, bias, eps, stats: bool):
    rows = rows_of(x)
    n, dim = rows.shape
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    saved = torch.empty((2, n), dtype=torch.float32, device=x.device) if stats else None
    if n:
        index = x.get_device()
        with on_device(index):
            _lib.check("rfm_layer_norm_forward", _lib.load().rfm_layer_norm_forward(
                rows.data_ptr(), row_stride(rows), weight.data_ptr() if weight is not None else None,
                bias.data_ptr() if bias is not None else None, out.data_ptr(),
                saved.data_ptr() if stats else None, saved.data_ptr() + 4 * n if stats else None, n, dim, eps,
                DTYPES[x.dtype], _param_code(x, weight, bias), raw_stream(index)))
    return out, rows, saved


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        out, rows, saved = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, saved)
        ctx.shape, ctx.param = x.shape, _param_code(x, weight, bias)
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else None
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weight, saved = ctx.saved_tensors
        n, dim = rows.shape
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        device = rows.device
        grad_x = torch.empty(ctx.shape, dtype=rows.dtype, device=device) if need_x else None
        grad_w = torch.empty(dim, dtype=ctx.param_dtype, device=device) if need_w else None
        grad_b = torch.empty(dim, dtype=ctx.param_dtype, device=device) if need_b else None
        g = rows_of(grad)
        lib = _lib.load()
        index = rows.get_device()
        with on_device(index):
            size = int(lib.rfm_layer_norm_workspace_bytes(n, dim)) if need_w or need_b else 0
            work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
            _lib.check("rfm_layer_norm_backward", lib.rfm_layer_norm_backward(
                rows.data_ptr(), row_stride(rows), weight.data_ptr() if weight is not None else None,
                saved.data_ptr(), saved.data_ptr() + 4 * n, g.data_ptr(), row_stride(g),
                grad_x.data_ptr() if need_x else None, grad_w.data_ptr() if need_w else None,
                grad_b.data_ptr() if need_b else None, n, dim, DTYPES[rows.dtype], ctx.param,
                work.data_ptr() if size else None, size, raw_stream(index)))
        return grad_x, grad_w, grad_b, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    ``x`` ``[..., D]`` float32, bfloat16 or float16, any leading shape and strides (rows whose elements
    are not adjacent are copied first); ``weight`` and ``bias`` ``[D]`` of ``x``'s type or float32, both of
    one type, either of them None.  Returns ``x``'s shape and type, contiguous, differentiable (once) in
    all three.
    """
    require_cuda(x, "x", "layer_norm")
    if x.dtype not in DTYPES:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs a last dimension of at least one element")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.device != x.device or p.shape != x.shape[-1:]:
            raise ValueError(f"{name} must have shape [{x.shape[-1]}] on x's device")
        if p.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be float32 or of x's type, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one type")
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
