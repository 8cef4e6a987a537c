"""GPU tests of the embedding, the norm and the loss where something records what is called: torch.jit.trace and tracers into fx graphs see torch's operations, and these
are launches."""

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]    # of tracing, and of torch.jit itself

DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(params=["nodes", "python"], autouse=True)
def host(request, monkeypatch):
    """Every test through the C++ calls and nodes, and through the Python ones that stand in for them."""
    from flashoptim_amd import _autograd

    _autograd.bind()
    assert _autograd.rms_norm and _autograd.rms_norm_mxfp4 and _autograd.embedding and _autograd.linear_cross_entropy
    if request.param == "python":
        for name in ("rms_norm", "rms_norm_mxfp4", "embedding", "linear_cross_entropy"):
            monkeypatch.setattr(_autograd, name, None)
    return request.param


def _fo():
    import flashoptim_amd

    return flashoptim_amd


def _calls():
    """Functions of tensors, with two sets of operands for each."""
    fo = _fo()
    g = torch.Generator(device=DEV).manual_seed(1)

    def some(*shapes):
        return [tuple(torch.randn(*s, generator=g, device=DEV).to(BF16) if isinstance(s, tuple) else torch.randint(0, 33, (s, 3), generator=g, device=DEV) for s in shapes)
                for _ in range(2)]

    yield "embedding", lambda t, w: fo.embedding(t, w, scale=2.0, padding_idx=-3) * 2, some(5, (33, 40))
    yield "norm", lambda x: fo.rms_norm(x) * 2, some((5, 3, 40))
    yield "norm with a weight", lambda x, w: fo.rms_norm(x, w), some((6, 40), (40,))
    yield "norm with a residual", lambda x, w, r: fo.rms_norm(x * 2, w, r), some((6, 40), (40,), (6, 40))
    yield "loss", lambda x, w, t: fo.linear_cross_entropy(x, w, t), some((5, 3, 40), (33, 40), 5)
    yield "losses", lambda x, w, t: fo.linear_cross_entropy(x, w, t, reduction="none", label_smoothing=0.1) * 2, some((5, 3, 40), (33, 40), 5)
    yield "modules", torch.nn.Sequential(fo.FlashEmbedding(33, 40, device=DEV, dtype=BF16), fo.FlashRMSNorm(40, device=DEV, dtype=BF16)), some(5)


def _tuple(out):
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("gradients", [False, True])
def test_traces_compute(gradients):
    for what, call, (first, second) in _calls():
        if gradients:
            first, second = (tuple(t.requires_grad_() if t.is_floating_point() else t for t in ts) for ts in (first, second))
        traced = torch.jit.trace(call, first, check_trace=False)
        for operands in (first, second, first):
            garbage = [torch.full((100000,), float("nan"), device=DEV) for _ in range(3)]    # what an output that nobody writes would be made of
            del garbage
            got, want = _tuple(traced(*operands)), _tuple(call(*operands))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), what
            leaves = [t for t in operands if t.is_floating_point()]
            if gradients and leaves:
                got, want = (torch.autograd.grad(sum((o.float() ** 2).sum() for o in outs), leaves) for outs in (got, want))
                assert all(torch.equal(a, b) for a, b in zip(got, want)), what


def test_a_trace_checks_the_call_it_records():
    fo = _fo()
    x = torch.randn(3, 8, device=DEV)
    with pytest.raises(ValueError):
        torch.jit.trace(lambda x: fo.rms_norm(x, torch.ones(7, device=DEV)), (x,), check_trace=False)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda x: fo.rms_norm_mxfp4(x).codes, (x,), check_trace=False)


@pytest.mark.parametrize("how", [dict(), dict(pre_dispatch=True)], ids=str)
def test_fx_graphs_are_refused(how):
    from torch.fx.experimental.proxy_tensor import make_fx

    fo = _fo()
    for what, call, (operands, _) in _calls():
        with pytest.raises(NotImplementedError, match="fx graph"):
            make_fx(call, **how)(*operands)
    with pytest.raises(NotImplementedError, match="fx graph"):
        make_fx(lambda x: fo.rms_norm_mxfp4(x).codes, **how)(torch.randn(3, 8, device=DEV))


def test_modes_that_only_look_on():
    from torch.utils.flop_counter import FlopCounterMode

    for what, call, (operands, _) in _calls():
        want = _tuple(call(*operands))
        with FlopCounterMode(display=False):
            got = _tuple(call(*operands))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), what
