"""Loads the native torch binding of the block operators (csrc/torch_binding.cpp,
built in-tree as lib/mlpk_torch.so).  Loading needs no GPU; there is no fallback:
if it is missing, the operators raise."""
from __future__ import annotations

import importlib.util
import os

from . import _lib

PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "mlpk_torch.so")
_module = None


def native():
    global _module
    if _module is None:
        if not os.path.exists(PATH):
            raise RuntimeError(f"{PATH} not found: build it with `python -m mlp_megakernel_b200.build` "
                               "(there is no CPU fallback)")
        _lib.lib()  # the library it calls
        spec = importlib.util.spec_from_file_location("mlpk_torch", PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _module = module
    return _module
