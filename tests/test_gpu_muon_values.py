"""GPU tests of single values on their way through the Muon step."""

import pytest
import torch
import torch.nn as nn

from tests.test_gpu_muon import DEV, _muon

pytestmark = pytest.mark.gpu


def test_momentum_codes_stand_for_what_dequantize_reads():
    """Every code, through one step that moves weights of zero along momentum codes, and through the same step with the momentum held in fp32 as
    `dequantize` gives it: to the bit.  (16 x 16 runs in fp32, and with coefficients (1, 0, 0) the step is the normalised momentum.)"""
    from flashoptim_amd.kernels import dequantize

    codes = torch.arange(256, device=DEV).to(torch.uint8).view(torch.int8).view(16, 16)
    codes[8, 0] = 0    # -128, which no quantiser writes
    scales = torch.tensor([1.0, 0.5, 3.0, 1e-3, 7.0, 0.1, 2.0, 1.0], device=DEV, dtype=torch.float16)
    moved = []
    for quantize in (True, False):
        weight = nn.Parameter(torch.zeros(16, 16, device=DEV))
        opt = _muon([weight], lr=1.0, weight_decay=0.0, nesterov=False, ns_steps=1, ns_coefficients=(1.0, 0.0, 0.0), master_weight_bits=None,
                    quantize=quantize)
        weight.grad = torch.zeros_like(weight)
        opt.step()
        assert not weight.any()
        held = opt.state[weight]["momentum_buffer"]
        if quantize:
            held.quantized.copy_(codes)
            held.scales.copy_(scales)
        else:
            held.data.copy_(dequantize(codes, scales))
        opt.step()
        moved.append(weight.detach().clone())
    assert moved[1].count_nonzero() >= 250
    assert torch.equal(moved[0], moved[1]), (moved[0] != moved[1]).sum().item()
