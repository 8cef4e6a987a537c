"""What the Python side of the matrix operators hands to the library, seen on the CPU: the library is a stand-in."""

import contextlib
import weakref

import pytest
import torch

import flashoptim_amd as fo
from flashoptim_amd import mxfp4


class _Library:
    """Stands in for the native library: notes what is alive when an entry is called, and does nothing."""

    def __init__(self, alive):
        self.alive, self.seen = alive, []

    def __getattr__(self, name):
        def entry(*args):
            self.seen.append((name, [ref() is not None for ref in self.alive], args))
            return 0

        return entry


def _without_device(monkeypatch):
    """Calls go up to the library on host tensors; returns the library and weak references to what `mxfp4` allocates."""
    made = []

    class Torch:
        def __getattr__(self, name):
            return getattr(torch, name)

        @staticmethod
        def empty(*args, **kwargs):
            t = torch.empty(*args, **kwargs)
            made.append(weakref.ref(t))
            return t

    library = _Library(made)
    monkeypatch.setattr(mxfp4, "torch", Torch())
    monkeypatch.setattr(mxfp4._native, "lib", lambda: library)
    monkeypatch.setattr(mxfp4._native, "device_guard", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(mxfp4._native, "current_stream_ptr", lambda device: None)
    monkeypatch.setattr(mxfp4.kernels, "_require_device", lambda *args: None)
    return library, made


@pytest.mark.parametrize("tokens,inner", [(1, 128), (16, 4096), (64, 14336)])
def test_memory_of_the_product_for_few_rows_is_held_over_the_call(monkeypatch, tokens, inner):
    """The result, and the workspace where more rows' blocks than the product quantises itself need one."""
    library, made = _without_device(monkeypatch)
    weight = fo.MXFP4Tensor(torch.zeros((5, inner // 2), dtype=torch.uint8), torch.zeros((5, inner // 32), dtype=torch.uint8), (5, inner))
    mxfp4._tokens(torch.zeros(tokens, inner), weight, torch.bfloat16)
    (name, alive, args), = library.seen
    needs = tokens * inner // 128 > mxfp4._RAW_BLOCKS
    assert name == "fo_mxfp4_tokens" and alive == [True] * (2 if needs else 1)
    assert (args[-3] is not None) == needs and args[-2] == (tokens * inner // 128 * 68 if needs else 0)
