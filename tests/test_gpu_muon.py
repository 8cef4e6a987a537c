"""GPU tests of the Newton-Schulz iteration and of FlashMuon against plain computations in 64 bits.

What they allow, from the kernels' arithmetic:
* the iteration multiplies fp16 parts, whose values are off by up to 2^-11 of themselves; such roundings of S, of its polynomial and
  of X meet in every step, the later steps shrink what the earlier ones left of it.  Four of them, ``ITERATION = 2^-9`` of the
  result's norm, bound the sum;
* a bf16 result is rounded once more, by up to 2^-8 of each element (half a step of eight bits);
* momentum codes follow the package's quantiser (tests/parity.py); a master weight moves by what the iteration
  gives and is rounded to one unit of its precision, plus 2^-23 of the weight for the fp32 steps on the way there.
"""

import copy
import warnings

import pytest
import torch
import torch.nn as nn

from oracle import torch_oracle as T
from tests import parity

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ITERATION = 2.0 ** -9
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _fo():
    import flashoptim_amd

    return flashoptim_amd


def _iterate(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The definition, in float64."""
    a, b, c = coefficients
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2)
    x = x.contiguous() / (x.square().sum((-1, -2), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-1, -2) if tall else x


def _matrices(*shape, seed=0, size=1.0, dtype=torch.float32):
    """A few strong directions above noise."""
    g = torch.Generator().manual_seed(seed)
    rows, cols = shape[-2:]
    strong = max(1, min(rows, cols) // 16)
    left = torch.randn(*shape[:-2], rows, strong, generator=g)
    right = torch.randn(*shape[:-2], strong, cols, generator=g)
    noise = torch.randn(shape, generator=g)
    return (size * (left @ right / strong ** 0.5 + 0.25 * noise)).to(dtype).to(DEV)


def _check(got, want, what):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape, what
    off = ((got.double() - want).abs() - 2.0 ** -8 * want.abs()).clamp(min=0.0)
    for one_off, one in zip(off.reshape(-1, *off.shape[-2:]), want.reshape(-1, *want.shape[-2:])):
        assert float(one_off.norm()) <= 1.01 * ITERATION * float(one.norm()), what


# ------------------------------------------------------------------------------------------------ the iteration


SHAPES = [
    (1, 1, 1), (4, 1, 1), (2, 1, 500), (2, 700, 1), (3, 2, 3), (3, 100, 37), (5, 33, 65), (4, 17, 900), (1, 900, 17),
    (3, 128, 128), (1, 128, 256), (2, 256, 128),                                 # the most that one workgroup holds
    (1, 129, 256), (1, 128, 257), (2, 130, 131), (1, 300, 600), (2, 250, 1000), (2, 513, 1025),
    (1, 640, 640), (1, 700, 1100), (1, 1100, 700), (1, 1000, 2730), (1, 1536, 1024), (1, 1535, 1024),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_iteration_against_float64(shape, dtype):
    x = _matrices(*shape, seed=sum(shape), dtype=dtype)
    _check(_fo().newton_schulz(x), _iterate(x), (shape, dtype))


@pytest.mark.parametrize("shape", [(1, 40, 9000), (1, 9000, 40), (3, 130, 5000), (1, 600, 8000), (1, 8000, 600), (2, 64, 20011), (1, 16, 65536), (1, 65536, 3),
                                   (40, 65, 4097), (1, 330, 14336)])
def test_long_matrices_against_float64(shape):
    """S comes as a sum over parts of the long axis."""
    for steps in (1, 5):
        x = _matrices(*shape, seed=sum(shape), dtype=torch.bfloat16)
        _check(_fo().newton_schulz(x, steps=steps), _iterate(x, steps), (shape, steps))


@pytest.mark.parametrize("steps,coefficients", [(1, COEFFICIENTS), (2, COEFFICIENTS), (3, COEFFICIENTS), (4, (2.0, -1.5, 0.5)),
                                                (2, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375))])
@pytest.mark.parametrize("shape", [(2, 60, 90), (2, 300, 310), (1, 600, 1300), (1, 1300, 600)])
def test_steps_and_coefficients(shape, steps, coefficients):
    x = _matrices(*shape, seed=steps)
    got = _fo().newton_schulz(x, steps=steps, coefficients=coefficients)
    _check(got, _iterate(x, steps, coefficients), (shape, steps, coefficients))


@pytest.mark.parametrize("size", [1e-12, 1e-6, 1.0, 1e4, 1e15])
@pytest.mark.parametrize("shape", [(60, 90), (300, 700)])
def test_magnitude_does_not_matter(shape, size):
    x = _matrices(*shape, seed=3, size=size)
    _check(_fo().newton_schulz(x, eps=0.0), _iterate(x, eps=0.0), (shape, size))


@pytest.mark.parametrize("eps", [0.0, 1e-7, 10.0])
@pytest.mark.parametrize("shape", [(60, 90), (300, 700)])
def test_eps_is_added_to_the_norm(shape, eps):
    x = _matrices(*shape, seed=4, size=0.01)
    _check(_fo().newton_schulz(x, eps=eps), _iterate(x, eps=eps), (shape, eps))


@pytest.mark.parametrize("shape", [(1, 1), (100, 30), (130, 700), (1300, 600)])
def test_a_matrix_of_zeros_stays_one(shape):
    fo = _fo()
    x = torch.zeros(2, *shape, device=DEV)
    x[1] = _matrices(*shape, seed=5)
    got = fo.newton_schulz(x)
    assert not got[0].any()
    assert torch.equal(got[1], fo.newton_schulz(x[1]))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("shape", [(20, 30), (130, 700), (700, 130), (1300, 600)])
def test_a_value_that_is_not_finite_spoils_its_matrix_alone(shape, bad):
    fo = _fo()
    x = _matrices(3, *shape, seed=6)
    want = fo.newton_schulz(x)
    x[1, -1, shape[1] // 2] = bad
    got = fo.newton_schulz(x)
    assert got[1].isnan().all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(37, 100), (250, 333)])
def test_strides_and_offsets(rows, cols, dtype):
    """The result is that of the contiguous copy, whatever the input's layout, and the transpose's is the transpose of it."""
    fo = _fo()
    wide = _matrices(3, rows + 3, cols + 9, seed=7, dtype=dtype)
    for view in (wide[:, 1:1 + rows, 5:5 + cols], wide[::2, 2:2 + rows, 1:1 + cols], wide[:, :rows, 3:3 + cols].flip(0),
                 wide.transpose(0, 1)[:, :, 4:4 + cols][:rows].transpose(0, 1), wide[1, 3:, 9:], wide[0, :rows, :cols].expand(4, rows, cols)):
        want = fo.newton_schulz(view.contiguous())
        got = fo.newton_schulz(view)
        assert got.is_contiguous() and torch.equal(got, want)
        turned = fo.newton_schulz(view.transpose(-1, -2))
        assert turned.shape == view.transpose(-1, -2).shape and torch.equal(turned, want.transpose(-1, -2))
        turned = fo.newton_schulz(view.transpose(-1, -2).contiguous())
        _check(turned, _iterate(view.transpose(-1, -2)), "transposed")
    every_other = wide[:, ::2, ::2]
    assert torch.equal(fo.newton_schulz(every_other), fo.newton_schulz(every_other.contiguous()))
    stack = wide[:, :rows, :cols].contiguous().view(1, 3, rows, cols)
    assert torch.equal(fo.newton_schulz(stack), fo.newton_schulz(stack[0]).view(1, 3, rows, cols))
    assert torch.equal(fo.newton_schulz(torch._neg_view(stack[0])), fo.newton_schulz(-stack[0].clone()))


def test_stacks_of_any_length_equal_single_matrices(monkeypatch):
    from flashoptim_amd import muon

    fo = _fo()
    x = _matrices(7, 140, 200, seed=8)
    want = torch.stack([fo.newton_schulz(one) for one in x])
    assert torch.equal(fo.newton_schulz(x), want)
    monkeypatch.setattr(muon, "WORKSPACE_BYTES", 3 * muon._workspace_bytes((muon.FoMatrixShape * 1)(muon.FoMatrixShape(140, 200, 1, 0.0)), 1))
    assert torch.equal(fo.newton_schulz(x), want)   # in parts of three
    many = _matrices(5000, 3, 5, seed=9)
    _check(fo.newton_schulz(many), _iterate(many), "many")


@pytest.mark.parametrize("shape", [(0, 5, 7), (3, 0, 7), (3, 7, 0), (0, 0)])
def test_empty_stacks(shape):
    got = _fo().newton_schulz(torch.empty(shape, device=DEV))
    assert got.shape == shape and got.dtype == torch.bfloat16


def test_more_elements_than_32_bits_count():
    """32 x 33 copies of one matrix side by side have the singular values of that matrix, times one number, so the result is that
    of the one matrix, repeated."""
    fo = _fo()
    one = _matrices(2048, 1000, seed=10, dtype=torch.bfloat16)
    x = one.repeat(32, 33)
    assert x.numel() > 2 ** 31
    got = fo.newton_schulz(x, eps=0.0)
    want = _iterate(one, eps=0.0) / (32 * 33) ** 0.5
    for i, j in ((0, 0), (31, 0), (15, 17), (0, 32), (31, 32)):
        _check(got[i * 2048:(i + 1) * 2048, j * 1000:(j + 1) * 1000], want, (i, j))


def test_on_another_stream_and_repeatable():
    fo = _fo()
    x = _matrices(2, 500, 900, seed=11)
    want = fo.newton_schulz(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 1.0
        torch.cuda._sleep(2_000_000)
        y.add_(0.0)
        got = [fo.newton_schulz(y) for _ in range(3)]
    side.synchronize()
    for one in got:
        assert torch.equal(one, want)


def test_iteration_in_a_graph():
    fo = _fo()
    shapes = [(2, 60, 90), (2, 300, 700)]
    x = [_matrices(*s, seed=12) for s in shapes]
    for one in x:
        fo.newton_schulz(one)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [fo.newton_schulz(one) for one in x]
    for seed in range(3):
        for one, s in zip(x, shapes):
            one.copy_(_matrices(*s, seed=20 + seed))
        want = [fo.newton_schulz(one) for one in x]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_iteration_refuses():
    fo = _fo()
    x = torch.zeros(4, 5, device=DEV)
    with pytest.raises(NotImplementedError):
        fo.newton_schulz(x.cpu())
    for bad in (x.double(), x.to(torch.int32), x[0]):
        with pytest.raises(ValueError):
            fo.newton_schulz(bad)
    for steps in (0, -1, 100, 2.5):
        with pytest.raises(ValueError, match="steps"):
            fo.newton_schulz(x, steps=steps)
    for coefficients in ((1.0, 2.0), (1.0, 2.0, 3.0, 4.0), (1.0, float("nan"), 0.0), (float("inf"), 0.0, 0.0)):
        with pytest.raises(ValueError, match="coefficients"):
            fo.newton_schulz(x, coefficients=coefficients)
    for eps in (-1e-9, float("nan")):
        with pytest.raises(ValueError, match="epsilon"):
            fo.newton_schulz(x, eps=eps)
    with pytest.raises(ValueError, match="65536"):
        fo.newton_schulz(torch.zeros(65537, 1, device=DEV))


# ------------------------------------------------------------------------------------------------ the optimizer


def _muon(params, **kwargs):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")   # training without masters is remarked on
        return _fo().FlashMuon(params, **kwargs)


def _make(shapes, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [nn.Parameter((0.05 * torch.randn(s, generator=g)).to(dtype).to(DEV)) for s in shapes]


def _grads(params, seed, size=1e-2):
    for i, p in enumerate(params):
        p.grad = _matrices(*p.shape, seed=seed * 100 + i, size=size, dtype=p.dtype)


def _holder_tensors(state):
    out = {k: v for k, v in state.items() if isinstance(v, torch.Tensor)}
    buffer = state["momentum_buffer"]
    if buffer.is_quantized():
        out.update(codes=buffer.quantized, scales=buffer.scales)
    else:
        out.update(m=buffer.data)
    return out


def _momentum(state, quantize):
    if not quantize:
        return _holder_tensors(state)["m"].cpu().float()
    buffer = state["momentum_buffer"]
    n = buffer.quantized.numel()
    return T.dequantize_ref(buffer.quantized.cpu().reshape(-1), buffer.scales.cpu().reshape(-1)[:(n + 31) // 32]).view(buffer.quantized.shape)


def _factor(adjust, rows, cols):
    return 0.2 * max(rows, cols) ** 0.5 if adjust == "match_rms_adamw" else max(1.0, rows / cols) ** 0.5


PRECISIONS = [(torch.float32, None, True), (torch.float32, None, False), (torch.bfloat16, 24, True), (torch.bfloat16, 32, True),
              (torch.bfloat16, 24, False), (torch.bfloat16, None, True), (torch.float16, 32, True), (torch.float16, None, False),
              (torch.float16, 24, True)]
LAYER = [(64, 32), (1, 1), (33, 65), (250, 1000), (1000, 250), (130, 130), (1, 77), (300, 128), (1000, 640), (130, 130)]


@pytest.mark.parametrize("dtype,bits,quantize", PRECISIONS)
@pytest.mark.parametrize("hyper", [dict(lr=2e-2), dict(lr=1e-2, nesterov=False, weight_decay=0.0, adjust_lr_fn="match_rms_adamw"),
                                   dict(lr=5e-2, momentum=0.0, ns_steps=3, adjust_lr_fn="original")])
def test_step_against_float64(dtype, bits, quantize, hyper):
    params = _make(LAYER, dtype, 1)
    opt = _muon(params, master_weight_bits=bits, quantize=quantize, **hyper)
    lr, decay, mu = hyper["lr"], hyper.get("weight_decay", 0.1), hyper.get("momentum", 0.95)
    masters_before = [parity.master_value(p.detach().cpu().reshape(-1), None) for p in params]
    before = [torch.zeros(p.shape) for p in params]
    differ = 0
    for it in range(3):
        _grads(params, it)
        opt.step()
        for i, p in enumerate(params):
            what = (tuple(p.shape), it)
            state = opt.state[p]
            g, old = p.grad.cpu().float(), before[i]
            # the momentum, operation by operation as the kernels form it
            keep = torch.tensor(1.0) - torch.tensor(mu, dtype=torch.float32)
            new = (old * torch.tensor(mu, dtype=torch.float32) + g * keep)
            buffer = state["momentum_buffer"]
            if quantize:
                codes, scales = T.quantize_ref(new.reshape(-1))
                apart = (buffer.quantized.cpu().reshape(-1).int() - codes.int()).abs()
                assert int(apart.max()) <= 1, what
                differ += int(apart.sum())
                parity.check_scales(buffer.scales.reshape(-1)[:scales.numel()], scales, f"{what}: momentum scales")
            else:
                held = _holder_tensors(state)["m"].cpu()
                step = parity.ulp_of(new.to(dtype)).view(new.shape)
                assert bool(((held.double() - new.double()).abs() <= step).all()), what
            update = (g * keep + new * mu if hyper.get("nesterov", True) else new).to(DEV)
            direction = _iterate(update, hyper.get("ns_steps", 5)).cpu()
            moved = lr * _factor(hyper.get("adjust_lr_fn"), *p.shape) * direction.reshape(-1)
            want = masters_before[i] * (1.0 - lr * decay) - moved
            ecc = state.get("error_bits")
            narrow, code = p.detach().cpu().reshape(-1), None if ecc is None else ecc.cpu().reshape(-1)
            got = parity.master_value(narrow, code)
            # one unit of the master for its rounding (a weight near a power of two has the unit above it), fp32 on the way
            unit = parity.master_unit(narrow, code) + 2.0 ** -22 * masters_before[i].abs() + 2.0 ** -22 * moved.abs()
            off = ((got - want).abs() - unit).clamp(min=0.0)
            assert float(off.norm()) <= 1.01 * ITERATION * float(moved.norm()), what
            masters_before[i], before[i] = got, _momentum(state, quantize)
    assert differ <= parity.CODE_MISMATCH_FRACTION * 3 * sum(p.numel() for p in params)


def test_equal_gradients_take_equal_steps_whatever_shares_the_launch():
    """A matrix moves alike on its own, among others, in any order, and one parameter at a time."""
    shapes = [(250, 300), (64, 40), (700, 500), (250, 300), (40, 64), (1, 9), (70, 5000), (600, 4000), (5000, 70)]
    together = _make(shapes, torch.bfloat16, 2)
    alone = [nn.Parameter(p.detach().clone()) for p in together]
    one_by_one = [nn.Parameter(p.detach().clone()) for p in together]
    a = _muon(together, lr=1e-2)
    b = [_muon([p], lr=1e-2) for p in alone]
    c = _muon(one_by_one[::-1], lr=1e-2)
    for it in range(3):
        _grads(together, it)
        for p, q, r in zip(together, alone, one_by_one):
            q.grad, r.grad = p.grad.clone(), p.grad.clone()
        a.step()
        for p, opt in zip(one_by_one, b):
            opt.step()
            c.step_param(p)
        for p, q, r, opt in zip(together, alone, one_by_one, b):
            assert torch.equal(p, q) and torch.equal(p, r)
            sa, sb, sc = _holder_tensors(a.state[p]), _holder_tensors(opt.state[q]), _holder_tensors(c.state[r])
            assert sa.keys() == sb.keys() == sc.keys()
            for k in sa:
                assert parity.bits_equal(sa[k], sb[k]) and parity.bits_equal(sa[k], sc[k]), k


def test_more_shapes_than_a_launch_takes_and_lists_beyond_the_workspace(monkeypatch):
    from flashoptim_amd import muon

    shapes = [(5 + i, 7 + (i * 5) % 11) for i in range(40)] + [(130 + i, 140) for i in range(20)] + [(150, 140)] * 3
    pa, pb = _make(shapes, torch.bfloat16, 3), _make(shapes, torch.bfloat16, 3)
    _grads(pa, 1)
    _grads(pb, 1)
    _muon(pa, lr=1e-2).step()
    monkeypatch.setattr(muon, "WORKSPACE_BYTES", 2 << 20)   # two or three of the larger ones at a time
    _muon(pb, lr=1e-2).step()
    for a, b in zip(pa, pb):
        assert torch.equal(a, b), tuple(a.shape)


def test_parameters_without_gradient_and_without_elements_stay():
    params = _make([(30, 40), (0, 7), (200, 150), (9, 0)], torch.bfloat16, 4)
    opt = _muon(params, lr=1e-2)
    _grads(params, 1)
    params[2].grad = None
    before = [p.detach().clone() for p in params]
    opt.step()
    assert not torch.equal(params[0], before[0])
    assert all(torch.equal(p, b) for p, b in zip(params[1:], before[1:]))
    _grads(params, 2)
    opt.step()
    assert not torch.equal(params[2], before[2])


def test_a_gradient_of_zeros_only_decays():
    params = _make([(40, 30), (200, 300)], torch.float32, 5)
    opt = _muon(params, lr=1e-1, weight_decay=0.5, master_weight_bits=None)
    before = [p.detach().clone() for p in params]
    for p in params:
        p.grad = torch.zeros_like(p)
    opt.step()
    for p, b in zip(params, before):
        assert bool(((p - 0.95 * b).abs() <= 2.0 ** -22 * b.abs()).all())


def test_the_learning_rate_follows_its_group_and_its_schedule():
    params = _make([(40, 30), (200, 300)], torch.float32, 6)
    opt = _muon([dict(params=params[:1], lr=1e-2), dict(params=params[1:], lr=0.0)], weight_decay=0.0, master_weight_bits=None)
    before = [p.detach().clone() for p in params]
    _grads(params, 1)
    opt.step()
    assert not torch.equal(params[0], before[0]) and torch.equal(params[1], before[1])
    single = _make([(40, 30)], torch.float32, 6)
    opt = _muon(single, lr=1e-2, weight_decay=0.0, master_weight_bits=None)
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 1.0 if step == 0 else 0.0)
    for moves in (True, False):
        before = single[0].detach().clone()
        _grads(single, 2)
        opt.step()
        schedule.step()
        assert torch.equal(single[0], before) is not moves


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("compress", [False, True])
def test_resume_from_a_checkpoint(compress, dtype):
    """A compressed checkpoint goes on to the bit, save that scales of the momentum of bf16 weights pass through bf16 when it is
    loaded, and one without codes holds the momentum in bf16."""
    shapes = [(64, 32), (250, 300), (130, 700)]
    pa = _make(shapes, dtype, 7)
    oa = _muon(pa, lr=1e-2, compress_state_dict=compress)
    for it in range(2):
        _grads(pa, it)
        oa.step()
    pb = [nn.Parameter(p.detach().clone()) for p in pa]
    ob = _muon(pb, lr=1e-2, compress_state_dict=compress)
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    oc = copy.deepcopy(oa)
    pc = oc.param_groups[0]["params"]
    for p, q in zip(pa, pb):  # what a checkpoint holds is what goes on
        sa, sb = _holder_tensors(oa.state[p]), _holder_tensors(ob.state[q])
        if compress:
            for k in sa:
                if k == "scales" and dtype == torch.bfloat16:
                    assert bool(((sa[k] - sb[k]).abs() <= 2.0 ** -8 * sa[k]).all())
                else:
                    assert parity.bits_equal(sa[k], sb[k]), k
    for it in range(2, 4):
        _grads(pa, it)
        _grads(pb, it)
        _grads(pc, it)
        oa.step()
        ob.step()
        oc.step()
    for a, b, c in zip(pa, pb, pc):
        assert torch.equal(a, c)
        if compress and dtype == torch.float16:
            assert torch.equal(a, b)
        else:
            assert float((a - b).detach().float().norm()) <= 2e-2 * float(a.detach().float().norm())


def test_gradient_release_equals_stepping():
    fo = _fo()
    x = torch.randn(16, 128, device=DEV, dtype=torch.bfloat16)

    def model():
        torch.manual_seed(3)
        return nn.Sequential(nn.Linear(128, 256, bias=False), nn.ReLU(), nn.Linear(256, 300, bias=False)).to(DEV).to(torch.bfloat16)

    ma, mb = model(), model()
    oa, ob = _muon(ma.parameters(), lr=1e-2), _muon(mb.parameters(), lr=1e-2)
    handle = fo.enable_gradient_release(mb, ob)
    for _ in range(3):
        oa.zero_grad()
        ma(x).float().square().sum().backward()
        oa.step()
        mb(x).float().square().sum().backward()
        assert all(p.grad is None for p in mb.parameters())
    handle.remove()
    for a, b in zip(ma.parameters(), mb.parameters()):
        assert torch.equal(a, b)
        assert torch.equal(oa.state[a]["error_bits"], ob.state[b]["error_bits"])


def test_step_in_a_graph():
    shapes = [(64, 32), (250, 300), (700, 500)]
    pa, pb = _make(shapes, torch.bfloat16, 8), _make(shapes, torch.bfloat16, 8)
    oa, ob = _muon(pa, lr=1e-2), _muon(pb, lr=1e-2)
    _grads(pa, 0)
    static = [p.grad for p in pa]

    def feed(seed):
        _grads(pb, seed)
        for g, p in zip(static, pb):
            g.copy_(p.grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for it in range(2):
            feed(it)
            oa.step()
            ob.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    feed(2)
    with torch.cuda.graph(graph):
        oa.step()
    graph.replay()
    ob.step()
    for it in range(3, 6):
        feed(it)
        torch.cuda.synchronize()
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        for a, b in zip(pa, pb):
            assert torch.equal(a, b), (it, tuple(a.shape))


def test_it_trains():
    """Regression onto a random linear map: the loss falls to a hundredth."""
    torch.manual_seed(9)
    target = torch.randn(200, 150, device=DEV) / 150 ** 0.5
    weight = nn.Parameter(torch.zeros(200, 150, device=DEV, dtype=torch.bfloat16))
    opt = _muon([weight], lr=0.1, weight_decay=0.0)
    first = last = None
    for step in range(200):
        opt.param_groups[0]["lr"] = 0.1 * (1.0 - step / 200)
        x = torch.randn(256, 150, device=DEV)
        loss = (x @ (weight.float() - target).t()).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        first, last = first or loss.item(), loss.item()
    assert last < 0.01 * first, (first, last)


def test_optimizer_refuses():
    fo = _fo()
    weight = nn.Parameter(torch.zeros(4, 5, device=DEV, dtype=torch.bfloat16))
    for bad in (nn.Parameter(torch.zeros(4, device=DEV)), nn.Parameter(torch.zeros(2, 3, 4, device=DEV))):
        with pytest.raises(ValueError, match="matrices only"):
            fo.FlashMuon([weight, bad])
    with pytest.raises(ValueError, match="65536"):
        fo.FlashMuon([nn.Parameter(torch.zeros(65537, 1, device=DEV))])
    opt = fo.FlashMuon([weight])
    with pytest.raises(ValueError, match="matrices only"):
        opt.add_param_group(dict(params=[nn.Parameter(torch.zeros(4, device=DEV))]))
    assert len(opt.param_groups) == 1
    weight.grad = torch.zeros(5, 4, device=DEV, dtype=torch.bfloat16).t()
    with pytest.raises(RuntimeError):
        opt.step()


def test_check_numerics_raises_when_the_learning_rate_cannot_move_the_weights():
    fo = _fo()
    weight = nn.Parameter(torch.full((256, 256), 100.0, device=DEV, dtype=torch.bfloat16))
    opt = fo.FlashMuon([weight], lr=1e-7, master_weight_bits=24, check_numerics=True)
    weight.grad = _matrices(256, 256, seed=1, dtype=torch.bfloat16)
    with pytest.raises(fo.NumericsError):
        opt.step()
