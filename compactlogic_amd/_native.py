"""The C++ side of autograd (csrc/autograd.cpp), loaded on first use: `_native.load()`."""
from __future__ import annotations

import torch

from . import _capi, timing

_module = None


def load():
    """The extension module; raises where it is missing or was built for another torch."""
    global _module
    if _module is None:
        _capi.load()
        try:
            from . import _autograd
        except ImportError as e:
            raise _capi.CompactLogicError(
                f"the autograd extension cannot be loaded ({e}); build it with "
                "`python -m compactlogic_amd.build`") from e
        if not torch.__version__.startswith(_autograd.torch_version):
            raise _capi.CompactLogicError(
                f"the autograd extension was built for torch {_autograd.torch_version}, this is "
                f"{torch.__version__}: run `python -m compactlogic_amd.build`")
        timing.attach(_autograd)
        _module = _autograd
    return _module
