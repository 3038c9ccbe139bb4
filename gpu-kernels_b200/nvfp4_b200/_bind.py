"""The torch-facing binding of the 16-bit operators (csrc/torch_bind.cpp, built in-tree by
build.py): loads the extension and hands it the entry points of the loaded library.  There
is no fallback: without it, every call raises.
"""
import ctypes as C
import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (the extension links torch's libraries)

from ._lib import check, lib

PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_torch_bind.so")
_ENTRIES = ("nvfp4_linear", "nvfp4_linear_dgrad", "nvfp4_linear_wgrad", "nvfp4_activation_backward",
            "nvfp4_activation_backward_workspace_size", "nvfp4_moe_route", "nvfp4_moe_route_workspace_size",
            "nvfp4_moe_route_backward", "nvfp4_moe_dispatch", "nvfp4_moe_combine", "nvfp4_moe_combine_backward")


def _load():
    if not os.path.exists(PATH):
        raise ImportError(f"{PATH} is missing: build it with `python gpu-kernels_b200/build.py`")
    loader = importlib.machinery.ExtensionFileLoader("_torch_bind", PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_torch_bind", loader))
    loader.exec_module(module)
    module.bind(check, *(C.cast(getattr(lib(), name), C.c_void_p).value for name in _ENTRIES))
    return module


class _Lazy:
    """The extension's functions, loaded on the first one's use (importing the package needs
    no built library)."""

    def __getattr__(self, name):
        module = _load()
        for f in dir(module):
            if not f.startswith("_"):
                setattr(self, f, getattr(module, f))
        return getattr(module, name)


native = _Lazy()
