"""The native host side of the layer operators: the ``_host`` extension, built in-tree by
``python -m rfdetr_training_throughput_b200.build`` next to ``librfm.so``.  There is no fallback: where
it is missing, every operator that needs it raises."""

from __future__ import annotations

import importlib
from types import ModuleType

_host: ModuleType | None = None


def host() -> ModuleType:
    global _host
    if _host is None:
        import torch  # noqa: F401  (the extension's symbols resolve against torch's libraries)

        try:
            _host = importlib.import_module("._host", __package__)
        except ImportError as e:
            raise RuntimeError("the _host extension is not built; run `python -m "
                               "rfdetr_training_throughput_b200.build` (there is no fallback)") from e
    return _host
