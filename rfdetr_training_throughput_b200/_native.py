"""The native host side of the layer operators: the ``_host`` extension, built in-tree by
``python -m rfdetr_training_throughput_b200.build`` next to ``librfm.so``.  There is no fallback: where
it is missing, every operator that needs it raises."""

from __future__ import annotations

import importlib
from types import ModuleType

import torch
from torch.autograd import forward_ad

_host: ModuleType | None = None


def host() -> ModuleType:
    global _host
    if _host is None:
        try:
            _host = importlib.import_module("._host", __package__)
        except ImportError as e:
            raise RuntimeError("the _host extension is not built; run `python -m "
                               "rfdetr_training_throughput_b200.build` (there is no fallback)") from e
    return _host


def reaches_kernels(*tensors: torch.Tensor | None) -> bool:
    """Whether a module's call on these tensors may go past torch's dispatcher: they are plain CUDA tensors,
    and no tracer, compiler, function transform or forward-mode derivative has to see what happens to them."""
    if torch.compiler.is_compiling() or forward_ad._current_level >= 0:
        return False
    for t in tensors:
        if t is not None and (type(t) not in (torch.Tensor, torch.nn.Parameter) or not t.is_cuda):
            return False
    return not host().intercepted()
