"""GPU tests of single values on their way through the Muon step and the iteration."""

import pytest
import torch
import torch.nn as nn

from tests.test_gpu_muon import DEV, _check, _fo, _grads, _iterate, _matrices, _muon

pytestmark = pytest.mark.gpu


def test_momentum_codes_stand_for_what_dequantize_reads():
    """Every code, through one step that moves weights of zero along momentum codes, and through the same step with the momentum held in fp32 as
    `dequantize` gives it.  (16 x 16 runs in fp32, and with coefficients (1, 0, 0) the step is the normalised momentum.)  The quotient by 127 is off by
    2^-23 at most, y / (2 - |y|) makes 2^-22 of it, the norm can shift by as much, and the roundings of fp32 add less than that again: 2^-20."""
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
    assert bool(((moved[0] - moved[1]).abs() <= 2.0 ** -20 * moved[1].abs()).all())


@pytest.mark.parametrize("size", [1e-36, 1e-30, 1e-22, 1e19, 1e25, 1e33])
@pytest.mark.parametrize("shape", [(10, 12), (60, 90), (300, 700), (700, 300)])
def test_matrices_whose_squares_fp32_does_not_hold(shape, size):
    x = _matrices(*shape, seed=3, size=size)
    assert x.isfinite().all() and float(x.abs().max()) > 2.0 ** -126
    _check(_fo().newton_schulz(x, eps=0.0), _iterate(x, eps=0.0), (shape, size))


@pytest.mark.parametrize("size", [1e-22, 1e19, 1e25, 1e33])
@pytest.mark.parametrize("shape", [(10, 12), (60, 90), (300, 700)])
@pytest.mark.parametrize("dtype,quantize", [(torch.float32, False), (torch.bfloat16, False)])
def test_steps_along_gradients_whose_squares_fp32_does_not_hold(shape, size, dtype, quantize):
    weight = nn.Parameter(torch.zeros(shape, device=DEV, dtype=dtype))
    opt = _muon([weight], lr=1.0, weight_decay=0.0, momentum=0.0, master_weight_bits=None, eps=0.0, quantize=quantize)
    weight.grad = _matrices(*shape, seed=4, size=size, dtype=dtype)
    opt.step()
    factor = max(1.0, shape[0] / shape[1]) ** 0.5
    _check((-weight.detach() / factor).to(torch.bfloat16), _iterate(weight.grad, eps=0.0), (shape, size, dtype))


def _numerics(shapes, lr, bits=24):
    fo = _fo()
    params = [nn.Parameter(torch.full(s, 100.0, device=DEV, dtype=torch.bfloat16)) for s in shapes]
    opt = fo.FlashMuon(params, lr=lr, master_weight_bits=bits, check_numerics=True)
    _grads(params, 1)
    return opt, params


def test_check_numerics_judges_each_matrix_by_its_own_step():
    """A square matrix beside a long one, whose steps are 32 times smaller: a learning rate that moves either alone is taken for the two of them
    where each is fine, and refused, by the long one, where only that is not."""
    fo = _fo()
    square, long = (64, 64), (64, 65536)

    def refused(shapes, lr):
        opt, params = _numerics(shapes, lr)
        try:
            for _ in range(2):      # the second step goes by what the first one kept
                _grads(params, 1)
                opt.step()
        except fo.NumericsError as e:
            return str(e)
        return ""

    rates = [2.0 ** -k for k in range(-8, 24)]
    alone = {s: min(lr for lr in rates if not refused([s], lr)) for s in (square, long)}
    assert alone[long] == 32 * alone[square]
    assert not refused([square, long], alone[long])
    assert refused([square, long], alone[long] / 2)
    # the long one sits out: nothing about it matters
    opt, params = _numerics([square, long], alone[square])
    params[1].grad = None
    opt.step()
    params[0].grad = params[0].grad.clone()
    opt.step()
    # a group of its own, with its own learning rate
    params = [nn.Parameter(torch.full(s, 100.0, device=DEV, dtype=torch.bfloat16)) for s in (square, long)]
    opt = fo.FlashMuon([dict(params=params[:1], lr=alone[square]), dict(params=params[1:], lr=alone[long])], check_numerics=True)
    for _ in range(2):
        _grads(params, 1)
        opt.step()
    opt.param_groups[0]["lr"] /= 2
    with pytest.raises(fo.NumericsError):
        opt.step()


@pytest.mark.parametrize("bad", [dict(ns_coefficients=(1.5, -0.5)), dict(ns_coefficients=(1.0, float("inf"), 0.0)), dict(ns_steps=0), dict(ns_steps=2.5), dict(eps=-1.0),
                                 dict(momentum=1.0), dict(weight_decay=-0.1), dict(adjust_lr_fn="spectral")])
def test_groups_are_checked_like_the_constructor(bad):
    """What a group says for itself, in the constructor's list or added later."""
    fo = _fo()
    first, second = (nn.Parameter(torch.zeros(8, 8, device=DEV, dtype=torch.bfloat16)) for _ in range(2))
    with pytest.raises(ValueError):
        fo.FlashMuon([dict(params=[first], **bad)])
    opt = fo.FlashMuon([dict(params=[first], ns_steps=3.0, ns_coefficients=[1.5, -0.5, 0.0], adjust_lr_fn="match_rms_adamw")])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[second], **bad))
    assert len(opt.param_groups) == 1
    first.grad = torch.ones_like(first)
    opt.step()
    assert first.any()
