"""A matrix's result does not depend on what shares its launches, at sizes where the tiles of the products go by the company.

With 256 compute units the square products of one 2048-wide matrix run in 64 x 64 tiles and those of three in 128 x 128, of one
4096-wide matrix in 192 x 192 and of five in 256 x 256; the steps' products change theirs as well.  Everything is compared to the bit.
"""

import pytest
import torch
import torch.nn as nn

from tests import parity
from tests.test_gpu_muon import DEV, _fo, _grads, _holder_tensors, _iterate, _make, _matrices, _muon, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,count", [(2048, 3072, 3), (3072, 2048, 3), (1024, 1536, 12), (2100, 5000, 3)])
def test_a_stack_equals_its_matrices(rows, cols, count):
    fo = _fo()
    x = _matrices(count, rows, cols, seed=rows, dtype=torch.bfloat16)
    together = fo.newton_schulz(x)
    for i in range(count):
        assert torch.equal(together[i], fo.newton_schulz(x[i])), i


@pytest.mark.parametrize("steps", [1, 2, 5])
def test_a_stack_of_the_widest_tiles_equals_its_matrices(steps):
    fo = _fo()
    x = _matrices(5, 4096, 4608, seed=2, dtype=torch.bfloat16)
    together = fo.newton_schulz(x, steps=steps)
    for i in range(5):
        assert torch.equal(together[i], fo.newton_schulz(x[i], steps=steps)), i


@pytest.mark.parametrize("shape", [(2048, 3072), (3072, 2048)])
def test_a_stack_against_float64(shape):
    x = _matrices(3, *shape, seed=1, dtype=torch.bfloat16)
    _check(_fo().newton_schulz(x), _iterate(x), shape)


@pytest.mark.parametrize("shapes", [[(2048, 5632)] * 3, [(4096, 6400), (1024, 4096), (1024, 4096), (4096, 6400), (6400, 4096)]])
def test_parameters_together_and_one_at_a_time(shapes):
    """The second list is the wide matrices of a layer with grouped keys and values."""
    together = _make(shapes, torch.bfloat16, 2)
    single = [nn.Parameter(p.detach().clone()) for p in together]
    a, b = _muon(together, lr=1e-2), _muon(single, lr=1e-2)
    for it in range(2):
        _grads(together, it)
        for p, q in zip(together, single):
            q.grad = p.grad.clone()
        a.step()
        for q in single:
            b.step_param(q)
        for i, (p, q) in enumerate(zip(together, single)):
            assert torch.equal(p, q), (it, i)
            sa, sb = _holder_tensors(a.state[p]), _holder_tensors(b.state[q])
            assert sa.keys() == sb.keys() and all(parity.bits_equal(sa[k], sb[k]) for k in sa), (it, i)
