"""GPU tests of the embedding lookup and its gradient against 64 bits.

What they allow: the lookup is one product and one rounding, as in torch, so it is exact.  A row of the gradient is the sum of n rows in fp32
(n - 1 additions of at most 2^-24 of the magnitudes' sum each), a product (2^-24) and half a step of the type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


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


def _tokens(n, vocabulary, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), vocabulary - 1)
    if kind == "runs":      # a few tokens with long lists, their borders anywhere
        return torch.randint(0, max(1, vocabulary // 5), (n,), generator=g) % 3 * (vocabulary // 3)
    t = torch.randint(0, vocabulary, (n,), generator=g)
    if kind == "padded":
        t[torch.rand(n, generator=g) < 0.6] = 0
    return t


def _check_gradient(dw, tokens, dy, vocabulary, scale, padding, what):
    tokens, dy = tokens.to(DEV).long(), dy.double()
    ok = (tokens >= 0) & (tokens < vocabulary)
    if padding is not None:
        ok &= tokens != padding
    kept, rows = tokens[ok], dy[ok]
    want = torch.zeros(vocabulary, dy.shape[1], dtype=torch.float64, device=DEV).index_add_(0, kept, rows) * scale
    size = torch.zeros_like(want).index_add_(0, kept, rows.abs()) * abs(scale)
    n = torch.bincount(kept, minlength=vocabulary).double().unsqueeze(1)
    bound = n * 2.0 ** -24 * size
    bound = bound + HALF_STEP[dw.dtype] * (want.abs() + bound) + SMALLEST[dw.dtype]
    assert bool(((dw.double() - want).abs() <= bound).all()), what
    assert not dw[n.squeeze(1) == 0].any(), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 7, 8, 250, 512, 513, 1031])
def test_rows_and_their_gradient(width, dtype):
    fo = _fo()
    for n, vocabulary, kind, index, scale, padding in [
            (1, 1, "any", torch.int64, 1.0, None), (1, 1000, "any", torch.int32, 2.5, None), (63, 10, "any", torch.int64, 1.0, 3),
            (511, 300, "any", torch.int32, math.sqrt(width), None), (513, 20, "padded", torch.int64, -0.3, -20), (1500, 5003, "any", torch.int64, 1.0, 5002),
            (1500, 31, "one", torch.int64, 1.0, None), (1500, 31, "one", torch.int64, 1.0, 30), (2100, 30, "runs", torch.int32, 0.1, None)]:
        what = (width, dtype, n, vocabulary, kind)
        tokens = _tokens(n, vocabulary, kind, seed=n).to(DEV, index)
        g = torch.Generator(device=DEV).manual_seed(width)
        weight = torch.randn(vocabulary, width, generator=g, device=DEV).to(dtype).requires_grad_()
        dy = torch.randn(n, width, generator=g, device=DEV).to(dtype)
        y = fo.embedding(tokens, weight, scale=scale, padding_idx=padding)
        assert torch.equal(y, (weight.detach()[tokens.long()].float() * scale).to(dtype)), what
        (dw,) = torch.autograd.grad(y, weight, dy, retain_graph=True)
        _check_gradient(dw, tokens, dy, vocabulary, scale, None if padding is None else padding % vocabulary, what)
        assert torch.equal(dw, torch.autograd.grad(y, weight, dy)[0]), what
        with torch.no_grad():
            assert torch.equal(fo.embedding(tokens, weight, scale=scale), y), what


@pytest.mark.parametrize("n", [512, 8192, 8193, 70001, 140000])
@pytest.mark.parametrize("kind", ["any", "padded", "runs"])
def test_many_tokens(n, kind):
    """One, two and three levels of sorting, lists that cross windows."""
    fo = _fo()
    vocabulary, width = 1000, 24
    tokens = _tokens(n, vocabulary, kind, seed=n).to(DEV)
    weight = torch.randn(vocabulary, width, device=DEV, requires_grad=True)
    dy = torch.randn(n, width, device=DEV)
    (dw,) = torch.autograd.grad(fo.embedding(tokens, weight), weight, dy)
    _check_gradient(dw, tokens, dy, vocabulary, 1.0, None, (n, kind))


def test_the_order_of_summing_is_that_of_the_tokens():
    """A list within one window (sixteen neighbours of the sorted tokens, counted from their first) is a plain sum in fp32 from the first position to the
    last; here every list is one window."""
    fo = _fo()
    vocabulary, width = 200, 16
    g = torch.Generator().manual_seed(3)
    tokens = torch.arange(vocabulary).repeat_interleave(16)[torch.randperm(16 * vocabulary, generator=g)]
    dy = torch.randn(16 * vocabulary, width, generator=g) * torch.exp2(torch.randint(-12, 12, (16 * vocabulary, 1), generator=g).float())
    want = torch.zeros(vocabulary, width)
    for i, t in enumerate(tokens.tolist()):
        want[t] += dy[i]
    weight = torch.zeros(vocabulary, width, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(fo.embedding(tokens.to(DEV), weight), weight, dy.to(DEV))
    assert torch.equal(dw.cpu(), want)


def test_shapes_strides_and_neighbours():
    fo = _fo()
    wide = torch.randn(50, 40, device=DEV, dtype=torch.bfloat16)
    weight = wide[:, 3:34]
    tokens = torch.randint(0, 50, (4, 5, 6), device=DEV)
    assert torch.equal(fo.embedding(tokens.transpose(0, 2), weight), weight[tokens.transpose(0, 2)])
    assert torch.equal(fo.embedding(tokens, weight.t().contiguous().t()), weight[tokens])
    assert torch.equal(fo.embedding(tokens[0, 0, 0], weight), weight[tokens[0, 0, 0]])
    assert fo.embedding(tokens[:0], weight).shape == (0, 5, 6, 31)
    # gradients whose rows lie apart, that repeat one row, and of no tokens
    leaf = weight.detach().clone().requires_grad_()
    for dy in (torch.randn(120, 70, device=DEV).to(torch.bfloat16)[:, 5:36], torch.randn(1, 31, device=DEV).to(torch.bfloat16).expand(120, 31),
               torch.randn(31, 120, device=DEV).to(torch.bfloat16).t()):
        (dw,) = torch.autograd.grad(fo.embedding(tokens.view(-1), leaf), leaf, dy)
        _check_gradient(dw, tokens.view(-1), dy, 50, 1.0, None, "strides")
    (dw,) = torch.autograd.grad(fo.embedding(tokens[:0], leaf), leaf, torch.zeros(0, 5, 6, 31, device=DEV, dtype=torch.bfloat16))
    assert dw.shape == leaf.shape and not dw.any()


def test_tokens_outside_the_vocabulary():
    fo = _fo()
    weight = torch.randn(10, 20, device=DEV, requires_grad=True)
    tokens = torch.tensor([3, -1, 10, 9, 1 << 40, -(1 << 40), 3, (1 << 32) + 3], device=DEV)
    y = fo.embedding(tokens, weight)
    bad = torch.tensor([False, True, True, False, True, True, False, True], device=DEV)
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], weight.detach()[tokens[~bad]])
    dy = torch.randn(8, 20, device=DEV)
    _check_gradient(torch.autograd.grad(y, weight, dy)[0], tokens, dy, 10, 1.0, None, "outside")


def test_infinities_stay_in_their_rows():
    fo = _fo()
    weight = torch.randn(10, 20, device=DEV, requires_grad=True)
    tokens = torch.tensor([3, 4, 4, 5], device=DEV)
    dy = torch.ones(4, 20, device=DEV)
    dy[1, 2], dy[3, 0] = float("inf"), float("nan")
    (dw,) = torch.autograd.grad(fo.embedding(tokens, weight, padding_idx=5), weight, dy)
    assert dw[4, 2] == float("inf") and bool(dw.isfinite().sum() == 199) and not dw[5].any()


def test_offsets_beyond_32_bits():
    fo = _fo()
    vocabulary, width = 300000, 8200        # 2.5e9 values
    weight = torch.zeros(vocabulary, width, device=DEV, dtype=torch.bfloat16)
    tokens = torch.tensor([vocabulary - 1, 0, 262144, vocabulary - 1], device=DEV)
    weight[tokens] = torch.randn(4, width, device=DEV).to(torch.bfloat16)
    weight.requires_grad_()
    y = fo.embedding(tokens, weight)
    assert torch.equal(y, weight.detach()[tokens])
    dy = torch.randn(4, width, device=DEV).to(torch.bfloat16)
    (dw,) = torch.autograd.grad(y, weight, dy)
    assert torch.equal(dw[tokens[1:3]], dy[1:3]) and torch.equal(dw[-1], (dy[0].float() + dy[3].float()).to(torch.bfloat16))
    assert int((dw != 0).any(1).sum()) == 3


def test_gradient_against_differences():
    fo = _fo()
    tokens = torch.randint(0, 12, (40,), device=DEV)
    weight = torch.randn(12, 9, device=DEV, requires_grad=True)
    dy, direction = torch.randn(40, 9, device=DEV), torch.randn(12, 9, device=DEV)
    (dw,) = torch.autograd.grad(fo.embedding(tokens, weight, scale=1.7), weight, dy)
    with torch.no_grad():
        ends = [(fo.embedding(tokens, weight + h * direction, scale=1.7).double() * dy).sum() for h in (0.5, -0.5)]
    # the function is linear: what separates the two is fp32's rounding of 360 values of order 1
    assert abs(float((dw.double() * direction).sum() - (ends[0] - ends[1]))) < 1e-4


def test_captured_and_replayed():
    fo = _fo()
    tokens = torch.randint(0, 100, (1500,), device=DEV)
    weight = torch.randn(100, 64, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn(1500, 64, device=DEV).to(torch.bfloat16)

    def both():
        leaf = weight.detach().requires_grad_()
        y = fo.embedding(tokens, leaf)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = both()
    for seed in range(3):
        tokens.copy_(torch.randint(0, 100, (1500,), generator=torch.Generator().manual_seed(seed)))
        dy.copy_(torch.randn(1500, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want_y, want_dw = both()
        assert torch.equal(y, want_y) and torch.equal(dw, want_dw), seed


def test_module():
    fo = _fo()
    layer = fo.FlashEmbedding(30, 16, padding_idx=2, scale=4.0, device=DEV, dtype=torch.bfloat16)
    tokens = torch.randint(0, 30, (5, 7), device=DEV)
    y = layer(tokens)
    y.sum().backward()
    assert torch.equal(y.detach(), layer.weight.detach()[tokens] * 4.0) and not layer.weight[2].any() and not layer.weight.grad[2].any()
    assert "scale=4.0" in repr(layer) and list(layer.state_dict()) == ["weight"]


def test_refusals():
    fo = _fo()
    weight, tokens = torch.zeros(4, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for bad in (dict(tokens=tokens.float()), dict(tokens=tokens.to(torch.int16)), dict(tokens=tokens.cpu()), dict(tokens=[1, 2]), dict(weight=weight[0]), dict(weight=weight.double()),
                dict(weight=weight.int()), dict(scale=float("nan")), dict(scale=float("inf")), dict(padding_idx=4), dict(padding_idx=-5)):
        with pytest.raises(ValueError):
            fo.embedding(**{**dict(tokens=tokens, weight=weight), **bad})
    with pytest.raises(NotImplementedError):
        fo.embedding(tokens.cpu(), weight.cpu())
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            fo.embedding(tokens, torch.autograd.forward_ad.make_dual(weight, torch.ones_like(weight)))
    weight.requires_grad_()
    (dw,) = torch.autograd.grad(fo.embedding(tokens, weight).square().sum(), weight, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dw.sum(), weight)

def test_one_derivative_only(host):
    """A second one is refused, also where it is only a part of what is asked for, and whatever came in does not require a gradient."""
    fo = _fo()
    leaf = torch.randn(9, 40, device=DEV, requires_grad=True)
    out = fo.embedding(torch.tensor([1, 2], device=DEV), leaf)
    first = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (first.sum() + (leaf * leaf).sum()).backward()
    assert (out.grad_fn.name() == "EmbeddingBackward") == (host == "nodes")
