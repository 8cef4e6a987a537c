"""GPU tests of the matrix products in the tiles that large sizes run in, against 64 bits.

Which tile a product takes goes by its size and the compute units (256 here): next to each case stands the edge of its tile, and of the tile that finishes it
where it is cut into two launches, by rows or by columns.  Tolerances are those of the small sizes' tests.
"""

import pytest
import torch
import torch.nn as nn

from tests import parity
from tests.test_gpu_muon import ITERATION, _check, _factor, _iterate, _make, _matrices, _muon
from tests.test_gpu_mxfp4 import DEV, _check_product, _fo, _random

pytestmark = pytest.mark.gpu


def _held(q):
    """What a form stands for; that the forms are right is tested for themselves."""
    return q.dequantize(torch.float32).double()


@pytest.mark.parametrize("m,n,k", [(1126, 2697, 102),     # 128
                                   (1688, 4706, 101),     # 192
                                   (2441, 4923, 389),     # 256
                                   (4096, 4096, 512)])    # 256, one round of whole tiles
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
def test_product(m, n, k, out):
    fo = _fo()
    qa, qb = fo.mxfp4_quantize(_random(m, k, seed=m)), fo.mxfp4_quantize(_random(n, k, seed=n + 1))
    _check_product(fo.mxfp4_matmul(qa, qb, out), _held(qa), _held(qb), (m, n, k, out))


LAYERS = [(617, 2757, 508),      # both gradients in 128
          (522, 3295, 1816),     # 192
          (542, 3101, 3202),     # 256
          (1389, 1744, 3428),    # 128, then 64 by columns
          (1377, 1767, 3497),    # 128, then 64 by rows
          (2467, 1554, 3235),    # 192, then 64 by columns
          (2049, 1679, 3380),    # 192, then 64 by rows
          (2068, 3352, 3464),    # 256, then 128 by columns
          (2344, 3410, 2970),    # 256, then 128 by rows
          (4096, 4096, 14336)]   # the layer of an 8B-parameter transformer: output and gradients all cut


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,inner,outer", LAYERS)
def test_layer_and_its_gradients(tokens, inner, outer, dtype):
    fo = _fo()
    x, w, dy = (_random(*shape, dtype, seed=i, spread=False) for i, shape in enumerate(((tokens, inner), (outer, inner), (tokens, outer))))
    leaf, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fo.mxfp4_linear(leaf, weight)
    y.backward(dy)
    both = [tuple(map(_held, fo.mxfp4_quantize_both(t))) for t in (x, w, dy)]
    (x_rows, x_columns), (w_rows, w_columns), (dy_rows, dy_columns) = both
    for got, a, b, what in ((y.detach(), x_rows, w_rows, "y"), (leaf.grad, dy_rows, w_columns, "dx"), (weight.grad, dy_columns, x_columns, "dw")):
        assert got.dtype == dtype
        _check_product(got, a, b, (what, tokens, inner, outer))


MATRICES = [(836, 5880),      # steps in 128
            (1410, 5388),     # 192
            (1860, 5989),     # 256
            (1803, 5937),     # 128, then 64 by columns
            (1733, 5872),     # 128, then 64 by rows
            (2447, 4469),     # 192, then 64 by columns
            (2306, 4672),     # 192, then 64 by rows
            (2825, 5920),     # 192, then 128 by columns
            (2706, 5915),     # 256, then 64 by columns
            (2822, 5651),     # 256, then 64 by rows
            (4096, 4096),     # squares in 192, steps in 256, nothing merged
            (4096, 14336)]    # squares in 192, steps in 256, then 128 by columns


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("shape", MATRICES)
def test_iteration(shape, turned):
    shape = shape[::-1] if turned else shape
    x = _matrices(*shape, seed=sum(shape), dtype=torch.bfloat16)
    _check(_fo().newton_schulz(x), _iterate(x), shape)


@pytest.mark.parametrize("shape,count", [((4096, 4608), 5), ((2048, 3072), 12)])
def test_stacks(shape, count):
    """Squares in 256, those of the merged steps among them."""
    x = _matrices(count, *shape, seed=count, dtype=torch.bfloat16)
    got = _fo().newton_schulz(x)
    for i in (0, count // 2, count - 1):
        _check(got[i], _iterate(x[i]), (shape, i))


@pytest.mark.parametrize("dtype,bits", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, 24), (torch.bfloat16, 32), (torch.float16, 24), (torch.float16, 32)])
@pytest.mark.parametrize("shapes", [[(836, 5880)], [(1410, 5388)], [(5388, 1410)], [(5937, 1803)], [(2822, 5651)], [(4096, 4096)], [(4096, 4096), (1410, 5388), (4096, 4096)]])
def test_step(shapes, dtype, bits):
    """Without momentum the update is the gradient: what is left is the iteration and the weights' way along it, in every tile that writes them."""
    params = _make(shapes, dtype, 1)
    lr, decay = 2e-2, 0.1
    opt = _muon(params, master_weight_bits=bits, lr=lr, weight_decay=decay, momentum=0.0)
    before = [parity.master_value(p.detach().clone(), None) for p in params]
    for it in range(2):
        for i, p in enumerate(params):
            p.grad = _matrices(*p.shape, seed=10 * it + i, size=1e-2, dtype=dtype)
        opt.step()
        for i, p in enumerate(params):
            moved = lr * _factor(None, *p.shape) * _iterate(p.grad)
            want = before[i] * (1.0 - lr * decay) - moved
            narrow, code = p.detach(), opt.state[p].get("error_bits")
            got = parity.master_value(narrow, code)
            unit = parity.master_unit(narrow, code) + 2.0 ** -22 * before[i].abs() + 2.0 ** -22 * moved.abs()
            off = ((got - want).abs() - unit).clamp(min=0.0)
            assert float(off.norm()) <= 1.01 * ITERATION * float(moved.norm()), (shapes[i], it)
            before[i] = got.clone()
