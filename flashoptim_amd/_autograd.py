"""Loader of the optional C++ calls and autograd nodes (flashoptim_amd/hostscan/fo_autograd.cpp).

Its functions (``rms_norm``, ``rms_norm_mxfp4``, ``embedding``, ``linear_cross_entropy``) are None when the module has not been built (``make -C
flashoptim_amd/hostscan``) or was built against another torch; they give None for operands out of the ordinary, and until the HIP
library has been loaded.  The Python functions around them (norm.py, embed.py, loss.py) then do the same host work themselves, to the same bits.
``FLASHOPTIM_NO_HOSTSCAN=1`` keeps the Python path.
"""

from __future__ import annotations

import ctypes
import importlib.util
import os

from . import _native

rms_norm = None
rms_norm_mxfp4 = None
embedding = None
linear_cross_entropy = None

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_fo_autograd.so")
_module = None


def _load() -> None:
    global _module, rms_norm, rms_norm_mxfp4, embedding, linear_cross_entropy
    if os.environ.get("FLASHOPTIM_NO_HOSTSCAN", "").strip() not in ("", "0") or not os.path.exists(_PATH):
        return
    try:
        spec = importlib.util.spec_from_file_location("_fo_autograd", _PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except (ImportError, OSError):  # built against another torch or python
        return
    _module = module
    rms_norm, rms_norm_mxfp4 = module.rms_norm, module.rms_norm_mxfp4
    embedding, linear_cross_entropy = module.embedding, module.linear_cross_entropy


def library_path() -> str:
    return _PATH


def bind() -> None:
    """Hands the C entry points of the loaded HIP library to the module."""
    global _module
    if _module is None:
        return
    lib = _native.lib()
    names = [n for n in _native.SIGNATURES if n == "fo_last_error" or n.startswith(("fo_rms_norm", "fo_embedding", "fo_linear_cross_entropy"))]
    _module.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
    _module = None  # once


_load()
