"""What the layer operators (``norm``, ``optim``, ``linear``) share on the host: element type codes,
the current stream, and the device a call's launches go to."""

from __future__ import annotations

from contextlib import nullcontext

import torch

from . import _lib

#: torch dtype -> RFM_DTYPE_*.
DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}

_NO_GUARD = nullcontext()


def raw_stream(index: int) -> int:
    """The current stream of device ``index`` as the integer the C ABI takes."""
    return torch._C._cuda_getCurrentRawStream(index)


def on_device(index: int):
    """A context in which device ``index`` is current: the library launches on the current device."""
    return _NO_GUARD if index == torch.cuda.current_device() else torch.cuda.device(index)


def require_cuda(t: torch.Tensor, name: str, what: str) -> int:
    """The device index of ``t``; raises for host tensors."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor ({what} has no CPU path)")
    return t.get_device()


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, last]`` with a unit stride along the rows' elements and rows that do not
    overlap: a view where the layout allows, else a copy."""
    last = x.shape[-1]
    y = x.reshape(-1, last) if x.numel() else x.new_empty((x.shape[:-1].numel(), last))
    if y.dim() == 2 and y.numel() and ((last > 1 and y.stride(1) != 1) or (y.shape[0] > 1 and y.stride(0) < last)):
        y = y.contiguous()
    return y


def row_stride(y: torch.Tensor) -> int:
    """Elements between the rows of a ``rows_of`` result (any value will do for a single row)."""
    return y.stride(0) if y.shape[0] > 1 else y.shape[1]
