"""What the Python side of the matrix operators hands to the library, seen on the CPU: the library is a stand-in."""

import contextlib
import weakref

import pytest
import torch
import torch.autograd.forward_ad as fwd

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


def _held(rows, cols):
    return fo.MXFP4Tensor(torch.zeros((rows, cols // 2), dtype=torch.uint8), torch.zeros((rows, cols // 32), dtype=torch.uint8), (rows, cols))


@pytest.mark.parametrize("shape", [(3, 128), (100, 128), (2, 3, 128)])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused_and_not_answered_with_nothing(monkeypatch, shape, grad):
    """A tangent is neither carried on nor lost without a word, whatever the weight and also where no gradients are recorded."""
    library, _ = _without_device(monkeypatch)
    x, weight = torch.zeros(shape), torch.zeros(5, 128)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = fwd.make_dual(x, torch.ones(shape))
        for call in (lambda: fo.mxfp4_linear(dual, _held(5, 128)), lambda: fo.mxfp4_linear(dual, weight),
                     lambda: fo.mxfp4_linear(x, fwd.make_dual(weight, torch.ones(5, 128)))):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        assert not library.seen
        fo.mxfp4_linear(x, _held(5, 128))    # without a tangent a level means nothing
        assert library.seen


@pytest.mark.parametrize("way", ["no_grad", "inference", "detached", "frozen"])
def test_calls_without_gradients_ask_for_no_column_forms(monkeypatch, way):
    """What the backward pass would need is neither allocated nor made where none can follow, whatever the operands say of themselves."""
    library, made = _without_device(monkeypatch)
    layer = fo.MXFP4Linear(128, 256, bias=False)
    x = torch.zeros(100, 128)
    if way == "frozen":
        layer.weight.requires_grad_(False)
    with {"no_grad": torch.no_grad, "inference": torch.inference_mode}.get(way, contextlib.nullcontext)():
        if way in ("no_grad", "inference"):
            y = layer(x.requires_grad_())
        else:
            y = fo.mxfp4_linear(x, layer.weight.detach() if way == "detached" else layer.weight)
    (name, _, args), = library.seen
    assert name == "fo_mxfp4_linear_forward" and not y.requires_grad
    assert args[9:11] == (None, None)
    assert len(made) == 2    # the output and the workspace


def test_calls_with_gradients_ask_for_the_forms_that_they_need(monkeypatch):
    library, _ = _without_device(monkeypatch)
    for dx in (True, False):
        for dw in (True, False):
            if dx or dw:
                y = fo.mxfp4_linear(torch.zeros(100, 128, requires_grad=dx), torch.zeros(256, 128, requires_grad=dw))
                name, _, args = library.seen[-1]
                assert name == "fo_mxfp4_linear_forward" and y.requires_grad
                assert (args[9] is not None, args[10] is not None) == (dw, dx)
