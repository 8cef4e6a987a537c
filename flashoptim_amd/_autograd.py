"""Loader of the optional C++ calls and autograd nodes (flashoptim_amd/hostscan/fo_autograd.cpp).

Its functions (``rms_norm``, ``rms_norm_mxfp4``, ``embedding``, ``linear_cross_entropy``) are None when the module has not been built (``make -C
flashoptim_amd/hostscan``) or was built against another torch or another C interface; they give None for operands out of the ordinary, and until the HIP
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


def _called() -> dict:
    """The C entry points that the module calls, with the types that the binding passes, in the module's letters."""
    letters = {ctypes.c_void_p: "P", ctypes.c_char_p: "P", ctypes.c_float: "f", ctypes.c_double: "d", ctypes.c_int32: "i", ctypes.c_int64: "q"}
    names = [n for n in _native.SIGNATURES if n == "fo_last_error" or n.startswith(("fo_rms_norm", "fo_embedding", "fo_linear_cross_entropy"))]
    return {n: "".join(letters[t] for t in (_native.SIGNATURES[n][0], *_native.SIGNATURES[n][1])) for n in names}


def _agreed() -> dict:
    return {**_called(), "FO_LINEAR_CROSS_ENTROPY_KEPT": str(_native.LOSS_NUMBERS_A_TOKEN + 1)}


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
    if getattr(module, "kinds", None) != _agreed():  # left over from another version of the library
        return
    _module = module
    rms_norm, rms_norm_mxfp4 = module.rms_norm, module.rms_norm_mxfp4
    embedding, linear_cross_entropy = module.embedding, module.linear_cross_entropy


def library_path() -> str:
    return _PATH


def bind() -> None:
    """Hands the C entry points of the loaded HIP library to the module, once; of threads that come here together each does, the same ones."""
    global _module
    module = _module
    if module is None:
        return
    lib = _native.lib()
    module.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _called()})
    _module = None


_load()
