"""GPU tests of the MXFP4 layer under torch's modes of differentiation."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.test_gpu_mxfp4 import DEV, _fo, _random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 5, 100])
def test_forward_mode_is_refused(tokens):
    """Also on the short way that a decoding step's call takes."""
    fo = _fo()
    x, w = _random(tokens, 256, torch.bfloat16, seed=1), _random(40, 256, torch.bfloat16, seed=2)
    held = fo.mxfp4_quantize(w)
    want = fo.mxfp4_linear(x, held)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for weight in (held, w):
            with pytest.raises(NotImplementedError, match="forward"):
                fo.mxfp4_linear(dual, weight)
        assert torch.equal(fo.mxfp4_linear(x, held), want)
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda t: fo.mxfp4_linear(t, held), (x,), (torch.ones_like(x),))
