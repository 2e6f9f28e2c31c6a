"""The compiled host path (``csrc/autograd.cpp``): C++ autograd functions over the library's C entry points, for the operators
whose calls are short enough for Python's share to show.  The reference's counterpart are the pybind modules of its
``cpp_jit`` (cute_kernels/jit.py:63-89).

``functions_for(tensor)`` is the module for an eager call on a GPU tensor and None otherwise: while a graph is traced the
Python autograd functions with their ``cute::`` custom ops are used, and tensors elsewhere get their refusal there."""

from __future__ import annotations

import importlib.util
import os
import threading

import torch

from . import _C
from .utils.custom_op import is_cute_tracing


_MODULE = "cute_autograd"
_module = None
_lock = threading.Lock()


def _import(path: str):
    spec = importlib.util.spec_from_file_location(_MODULE, path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def load():
    """Import (building first if nothing is built) and connect it to the kernel library; errors are not hidden."""
    global _module
    if _module is not None:
        return _module
    with _lock:
        if _module is not None:
            return _module
        from . import _build

        if not os.path.exists(_build.AUTOGRAD_PATH):
            _build.build_autograd()
        _C.load_library()
        module = _import(_build.AUTOGRAD_PATH)
        # (the library's version says nothing of the signatures an older build of the module calls it with)
        built_for = getattr(module, "abi_version", None)
        if built_for != _C._ABI_VERSION:
            raise RuntimeError(
                f"cute_autograd.so was built for ABI version {built_for}, this package needs {_C._ABI_VERSION}: rebuild it"
            )
        module.load(_C.library_path(), _C._ABI_VERSION)
        _module = module
    return _module


def functions_for(tensor: torch.Tensor):
    if not tensor.is_cuda or torch.compiler.is_compiling() or is_cute_tracing():
        return None
    return _module or load()


def not_differentiable(*grads: torch.Tensor | None) -> tuple[torch.Tensor | None, ...]:
    """For the end of a Python autograd function's backward that computes its gradients in kernels: where a graph of the
    backward is asked for (``create_graph=True``), differentiating them again is an error on every way to the function's
    inputs.  (torch's ``once_differentiable`` puts its error beside those ways: a sum of which another term can be
    differentiated misses this one without a word.)  While a graph is traced torch.compile itself refuses a second
    derivative."""
    if torch.compiler.is_compiling() or not torch.is_grad_enabled():
        return grads
    return tuple(load().not_differentiable(list(grads)))
