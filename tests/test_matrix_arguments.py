"""What the matrix operators refuse before any device work, through their C entry points and through Python, and what their
Python side computes on its own."""

import ctypes

import pytest
import torch
import torch.nn as nn

import flashoptim_amd as fo
from flashoptim_amd import _native, mxfp4, muon
from flashoptim_amd._native import FoMatrixShape

INVALID, UNSUPPORTED = -1, -2
THREE = (ctypes.c_float * 3)(1.0, 2.0, 3.0)
SOME = 1 << 20    # an address that no call here gets to use


def _shapes(*shapes):
    return (FoMatrixShape * len(shapes))(*[FoMatrixShape(r, c, n, 0.0) for r, c, n in shapes])


def test_iteration_checks_its_arguments():
    lib = _native.lib()

    def call(x=SOME, dtype=1, count=1, rows=4, cols=5, result=SOME, steps=5, coefficients=THREE, eps=1e-7, workspace=SOME, size=1 << 30):
        return lib.fo_newton_schulz(x, dtype, count, rows, cols, rows * cols, cols, result, steps, coefficients, eps, workspace, size, None)

    for bad in (dict(dtype=3), dict(dtype=-1), dict(count=-1), dict(rows=-1), dict(cols=-1), dict(count=1 << 31), dict(steps=0), dict(coefficients=None),
                dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(result=None), dict(workspace=None), dict(workspace=SOME + 128), dict(size=100)):
        assert call(**bad) == INVALID, bad
        assert lib.fo_last_error()
    assert call(rows=65537) == UNSUPPORTED and call(cols=65537) == UNSUPPORTED
    for nothing in (dict(count=0), dict(rows=0), dict(cols=0)):
        assert call(x=None, result=None, workspace=None, size=0, **nothing) == 0


def test_step_checks_its_arguments():
    lib = _native.lib()

    def call(matrices=SOME, shapes=_shapes((4, 5, 1)), n=1, dtype=1, ecc=1, steps=5, coefficients=THREE, eps=1e-7, workspace=SOME, size=1 << 30):
        return lib.fo_muon_step(matrices, shapes, n, dtype, ecc, 1, 1.0, 0.95, 1, steps, coefficients, eps, workspace, size, None)

    for bad in (dict(dtype=3), dict(ecc=3), dict(ecc=-1), dict(steps=0), dict(coefficients=None), dict(eps=-1.0), dict(n=-1), dict(shapes=None),
                dict(matrices=None), dict(workspace=None), dict(workspace=SOME + 1), dict(size=0), dict(shapes=_shapes((-1, 5, 1))), dict(shapes=_shapes((1, 5, -1)))):
        assert call(**bad) == INVALID, bad
    assert call(dtype=0, ecc=1) == UNSUPPORTED and call(shapes=_shapes((4, 65537, 1))) == UNSUPPORTED
    assert call(n=0, shapes=None, matrices=None, workspace=None, size=0) == 0
    assert call(shapes=_shapes((0, 5, 1), (5, 0, 2), (3, 4, 0)), n=3, matrices=None, workspace=None, size=0) == 0


def test_workspace_is_what_the_matrices_take():
    lib = _native.lib()
    size = lambda *shapes: lib.fo_newton_schulz_workspace(_shapes(*shapes), len(shapes))
    assert size((0, 5, 3)) == 0 and lib.fo_newton_schulz_workspace(None, 0) == 0
    one = size((250, 1000, 1))
    assert one % 256 == 0 and size((250, 1000, 7)) == 7 * one
    assert size((250, 1000, 1), (64, 64, 2)) == one + size((64, 64, 2))
    # lists longer than a launch takes use the space again
    many = [(100 + i, 50, 1) for i in range(40)]
    assert size(*many) < sum(size(s) for s in many)
    assert size(*many) >= max(size(s) for s in many)
    assert size((1, 65537, 1)) == UNSUPPORTED and size((1, -1, 1)) == INVALID
    # square, the largest: four of its arrays and three squares beside them
    assert size((65536, 65536, 1)) > 10 * 65536 ** 2


def test_quantiser_checks_its_arguments():
    lib = _native.lib()

    def call(x=SOME, dtype=1, rows=4, cols=5, codes=SOME, scales=SOME, column_codes=SOME, column_scales=SOME):
        return lib.fo_mxfp4_quantize(x, dtype, rows, cols, cols, codes, scales, column_codes, column_scales, None)

    for bad in (dict(dtype=3), dict(rows=-1), dict(cols=-1), dict(x=None), dict(codes=None), dict(scales=None), dict(column_codes=None), dict(column_scales=None),
                dict(codes=None, scales=None, column_codes=None, column_scales=None), dict(codes=SOME + 8), dict(column_codes=SOME + 4)):
        assert call(**bad) == INVALID, bad
    assert call(rows=1 << 31) == UNSUPPORTED and call(rows=1 << 30, cols=1 << 30) == UNSUPPORTED
    assert call(rows=0) == 0 and call(cols=0, x=None) == 0

    def back(codes=SOME, scales=SOME, rows=4, cols=5, out=SOME, dtype=1):
        return lib.fo_mxfp4_dequantize(codes, scales, rows, cols, out, dtype, None)

    for bad in (dict(codes=None), dict(scales=None), dict(out=None), dict(dtype=5), dict(rows=-1), dict(codes=SOME + 2)):
        assert back(**bad) == INVALID, bad
    assert back(rows=1 << 30, cols=1 << 20) == UNSUPPORTED
    assert back(rows=0, codes=None) == 0


def test_products_check_their_arguments():
    lib = _native.lib()

    def product(a=SOME, sa=SOME, rows=4, b=SOME, sb=SOME, cols=5, inner=6, out=SOME, dtype=1):
        return lib.fo_mxfp4_product(a, sa, rows, b, sb, cols, inner, out, dtype, None)

    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(dtype=-1), dict(rows=-1), dict(inner=-1), dict(a=SOME + 8),
                dict(sb=SOME + 2)):
        assert product(**bad) == INVALID, bad
    assert product(inner=0) == UNSUPPORTED and product(inner=(1 << 24) + 1) == UNSUPPORTED
    assert product(rows=0, a=None) == 0 and product(cols=0) == 0

    def tokens(x=SOME, dtype=1, n=4, weight=SOME, scales=SOME, cols=5, inner=6, out=SOME, out_dtype=1, workspace=None, size=0):
        return lib.fo_mxfp4_tokens(x, dtype, n, inner, weight, scales, cols, inner, out, out_dtype, workspace, size, None)

    for bad in (dict(x=None), dict(dtype=4), dict(weight=None), dict(scales=None), dict(out=None), dict(out_dtype=4), dict(n=-1), dict(weight=SOME + 8),
                dict(n=64, inner=14336), dict(n=64, inner=14336, workspace=SOME, size=100), dict(n=64, inner=14336, workspace=SOME + 8, size=1 << 30)):
        assert tokens(**bad) == INVALID, bad
    assert tokens(n=65) == UNSUPPORTED and tokens(inner=0) == UNSUPPORTED
    assert tokens(n=0) == 0 and tokens(cols=0) == 0
    assert lib.fo_mxfp4_tokens_workspace(1, 14336) == 0 and lib.fo_mxfp4_tokens_workspace(64, 14336) == 64 * 112 * 68


def test_layer_checks_its_arguments():
    lib = _native.lib()

    def forward(x=SOME, x_dtype=1, tokens=4, w=SOME, w_dtype=1, outer=5, inner=6, xc=SOME, wc=SOME, out=SOME, workspace=SOME, size=1 << 20):
        return lib.fo_mxfp4_linear_forward(x, x_dtype, tokens, inner, w, w_dtype, outer, inner, inner, xc, wc, out, workspace, size, None)

    for bad in (dict(x=None), dict(w=None), dict(out=None), dict(workspace=None), dict(x_dtype=7), dict(w_dtype=7), dict(tokens=-1), dict(size=100),
                dict(xc=SOME + 4), dict(wc=SOME + 4), dict(workspace=SOME + 4)):
        assert forward(**bad) == INVALID, bad
    for bad in (dict(tokens=0), dict(outer=0), dict(inner=0)):
        assert forward(**bad) == UNSUPPORTED, bad

    def backward(dy=SOME, dtype=1, tokens=4, outer=5, inner=6, xc=SOME, wc=SOME, dx=SOME, dw=SOME, dx_dtype=1, dw_dtype=1, workspace=SOME, size=1 << 20):
        return lib.fo_mxfp4_linear_backward(dy, dtype, tokens, outer, outer, inner, xc, wc, dx, dx_dtype, dw, dw_dtype, workspace, size, None)

    for bad in (dict(dy=None), dict(workspace=None), dict(xc=None), dict(wc=None), dict(dx=None), dict(dw=None), dict(dx=None, wc=None, dw=None, xc=None),
                dict(dtype=7), dict(dx_dtype=7), dict(dw_dtype=7), dict(size=100), dict(xc=SOME + 4)):
        assert backward(**bad) == INVALID, bad
    for bad in (dict(tokens=0), dict(outer=0), dict(inner=0)):
        assert backward(**bad) == UNSUPPORTED, bad


def test_sizes_that_python_computes_are_the_librarys():
    lib = _native.lib()
    for rows in (1, 3, 64, 1003):
        for cols in (1, 31, 128, 129, 2730, 14336):
            assert mxfp4._form_bytes(rows, cols) == lib.fo_mxfp4_form_bytes(rows, cols)
            if rows <= 64:
                blocks = rows * mxfp4._blocks(cols)
                assert lib.fo_mxfp4_tokens_workspace(rows, cols) == (0 if blocks <= mxfp4._RAW_BLOCKS else blocks * 68)


def test_hyperparameters_are_checked_before_the_device():
    p = [nn.Parameter(torch.zeros(4, 4))]
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(adjust_lr_fn="other"), dict(ns_steps=0), dict(ns_steps=100),
                dict(ns_coefficients=(1.0, 2.0)), dict(ns_coefficients=(1.0, 2.0, float("nan"))), dict(eps=-1.0), dict(master_weight_bits=16),
                dict(quantize=False, compress_state_dict=True)):
        with pytest.raises(ValueError):
            fo.FlashMuon(p, **bad)


def test_tensors_on_the_host_are_declined():
    x = torch.zeros(4, 5)
    for call in (lambda: fo.newton_schulz(x), lambda: fo.mxfp4_quantize(x), lambda: fo.mxfp4_quantize_both(x), lambda: fo.mxfp4_linear(x, x),
                 lambda: fo.mxfp4_linear(x, fo.MXFP4Tensor(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8), (3, 5)))):
        with pytest.raises(NotImplementedError):
            call()


def test_learning_rates_follow_the_shape():
    assert muon._update_factor(None, 400, 100) == 2.0 and muon._update_factor("original", 100, 400) == 1.0
    assert muon._update_factor("match_rms_adamw", 100, 400) == pytest.approx(4.0)


def test_public_names():
    for name in ("FlashMuon", "newton_schulz", "MXFP4Tensor", "MXFP4Linear", "mxfp4_quantize", "mxfp4_quantize_both", "mxfp4_dequantize", "mxfp4_matmul",
                 "mxfp4_linear"):
        assert name in fo.__all__ and hasattr(fo, name)
