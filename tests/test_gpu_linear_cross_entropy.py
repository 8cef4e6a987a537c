"""GPU tests of the cross entropy from hidden states and of its gradients against 64 bits.

What they allow, with u = 2^-24, S the largest sum of |x| |w| of a row's logits, k the values contracted:
* a logit is a sum of k products in fp32: (k u + 2^-23) S, as for the other matrix products; of fp32 operands, which are cut in
  parts, (2 k u + 2^-22) S;
* the log of the sum of exponentials has twice that, and 2^-16: exponents up to 2^7 times 2^-24 and the additions of at most 130 partial
  sums; the loss 2^-22 of itself besides;
* a probability p is off by p (twice the logits' error + 2^-16); G is rounded to the operands' type once (half a step; fp32's parts 2^-22);
  a gradient is a sum of such terms: their share of sum |G| |w|, and a contraction over n values n u + 2^-23 of it; then half a step of the type.
  fp16 does not hold probabilities below 2^-39 of the largest factor: 2^-40 of it times sum |w|.
"""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SMALLEST = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}
IGNORE = -100


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


def _slack(k, dtype):
    return 2 * k * 2.0 ** -24 + 2.0 ** -22 if dtype == F32 else k * 2.0 ** -24 + 2.0 ** -23


def _check(x, w, target, reduction, smoothing, upstream, loss, dx, dw, what):
    """loss, dx and dw (each may be None) of the call, with `upstream` the loss's gradient."""
    dtype, k, v = x.dtype, x.shape[1], w.shape[0]
    kept = target != IGNORE
    x64, w64, at = torch.where(kept.unsqueeze(1), x.double(), 0.0), w.double(), torch.where(kept, target, 0).long()
    z = x64 @ w64.t()
    e_z = _slack(k, dtype) * (x64.abs() @ w64.abs().t()).amax(1)
    lse = z.logsumexp(1)
    each = lse - (1 - smoothing) * z.gather(1, at.unsqueeze(1)).squeeze(1) - smoothing * z.mean(1)
    each = torch.where(kept, each, 0.0)
    e_each = torch.where(kept, 2 * e_z + 2.0 ** -16 + 2.0 ** -22 * each.abs(), 0.0)
    count = int(kept.sum())
    if loss is not None:
        assert loss.dtype == F32
        if reduction == "none":
            assert bool(((loss.double() - each).abs() <= e_each).all()), (what, "loss")
            assert not loss[~kept].any(), what
        else:
            over = count if reduction == "mean" else 1
            want, bound = float(each.sum()) / over, float(e_each.sum()) / over
            assert abs(float(loss) - want) <= bound + 2.0 ** -22 * abs(want), (what, "loss")
    factor = torch.where(kept, upstream.double().expand(target.shape), 0.0) / (count if reduction == "mean" else 1)
    p = torch.exp(z - lse.unsqueeze(1))
    g = p - smoothing / v
    g.scatter_add_(1, at.unsqueeze(1), torch.full_like(lse, smoothing - 1).unsqueeze(1))
    g *= factor.unsqueeze(1)
    size = p + smoothing / v
    size.scatter_add_(1, at.unsqueeze(1), torch.full_like(lse, 1 - smoothing).unsqueeze(1))
    size *= factor.abs().unsqueeze(1)
    error = (2 * e_z + 2.0 ** -16).unsqueeze(1) * p * factor.abs().unsqueeze(1) + max(HALF_STEP[dtype], 2.0 ** -22) * size
    if dtype == F16:
        error = error + 2.0 ** -40 * float(factor.abs().max())
    for got, left, off, right, n in ((dx, g, error, w64, v), (dw, g.t(), error.t(), x64, x.shape[0])):
        if got is None:
            continue
        want = left @ right
        bound = off @ right.abs() + (_slack(n, dtype)) * ((left.abs() + off) @ right.abs())
        bound = bound + HALF_STEP[dtype] * (want.abs() + bound) + SMALLEST[dtype]
        far = (got.double() - want).abs()
        assert got.dtype == dtype and bool((far <= bound).all()), (what, tuple(got.shape), float((far / bound).max()))


def _inputs(tokens, width, vocabulary, dtype, seed=0, ignored=0.0, index=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(vocabulary, width, generator=g, device=DEV) * width ** -0.5 * 1.5).to(dtype)
    target = torch.randint(0, vocabulary, (tokens,), generator=g, device=DEV)
    known = torch.rand(tokens, 1, generator=g, device=DEV) * 5.0
    x = (torch.randn(tokens, width, generator=g, device=DEV) + known * w[target].float()).to(dtype)
    target[torch.rand(tokens, generator=g, device=DEV) < ignored] = IGNORE
    return x.requires_grad_(), w.requires_grad_(), target.to(index)


def _both(tokens, width, vocabulary, dtype, reduction, smoothing=0.0, ignored=0.0, index=torch.int64):
    fo = _fo()
    what = (tokens, width, vocabulary, dtype, reduction, smoothing)
    x, w, target = _inputs(tokens, width, vocabulary, dtype, tokens + vocabulary, ignored, index)
    if reduction == "mean" and ignored:
        target[0] = 0
    loss = fo.linear_cross_entropy(x, w, target, reduction=reduction, label_smoothing=smoothing)
    upstream = torch.rand(tokens, device=DEV) - 0.3 if reduction == "none" else torch.tensor(0.7, device=DEV)
    dx, dw = torch.autograd.grad(loss, (x, w), upstream, retain_graph=True)
    _check(x.detach(), w.detach(), target, reduction, smoothing, upstream, loss.detach(), dx, dw, what)
    again = torch.autograd.grad(loss, (x, w), upstream)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]), what
    with torch.no_grad():
        assert torch.equal(fo.linear_cross_entropy(x, w, target, reduction=reduction, label_smoothing=smoothing), loss), what


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [1, 2, 31, 33, 64, 300])
def test_loss_and_gradients(tokens, dtype):
    for width, vocabulary, reduction, smoothing, ignored, index in [
            (1, 1, "mean", 0.0, 0.0, torch.int64), (8, 2, "none", 0.0, 0.3, torch.int32), (31, 63, "sum", 0.1, 0.3, torch.int64), (32, 64, "mean", 0.0, 0.0, torch.int32),
            (64, 65, "none", 0.3, 0.9, torch.int64), (100, 257, "mean", 0.0, 0.5, torch.int64), (520, 1000, "sum", 0.0, 0.0, torch.int64), (256, 5003, "mean", 1.0, 0.1, torch.int64)]:
        _both(tokens, width, vocabulary, dtype, reduction, smoothing, ignored, index)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [(1000, 1000, 4100), (2049, 96, 2000), (700, 2048, 700), (260, 4096, 9000)], ids=str)
def test_tiles_of_every_size(sizes, dtype):
    _both(*sizes, dtype, "mean", 0.1, 0.2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_vocabulary_in_pieces(dtype):
    """More than 2^27 logits (2^27 / 6 in fp32): the gradient goes piece by piece, dx through fp32 sums."""
    _both(*((2048, 40, 70001) if dtype == BF16 else (1024, 40, 50001)), dtype, "mean", 0.05, 0.1)


def test_tokens_in_blocks():
    _both(40001, 24, 130, BF16, "mean", 0.0, 0.3)


def test_strides():
    fo = _fo()
    for dtype in (F32, BF16, F16):
        wide_x, wide_w = torch.randn(40, 300, device=DEV).to(dtype), torch.randn(70, 301, device=DEV).to(dtype)
        target = torch.randint(0, 70, (40,), device=DEV)
        for cut in (slice(0, 64), slice(8, 72), slice(3, 67), slice(5, 200)):
            views = [wide_x[:, cut].detach().requires_grad_(), wide_w[:, cut].detach().requires_grad_()]
            whole = [t.detach().contiguous().requires_grad_() for t in views]
            a, b = (fo.linear_cross_entropy(*t, target) for t in (views, whole))
            assert torch.equal(a, b)
            for p, q in zip(torch.autograd.grad(a, views), torch.autograd.grad(b, whole)):
                assert torch.equal(p, q), (dtype, cut)
        x, w = wide_x[:, :64], wide_w[:, :64]
        same = fo.linear_cross_entropy(x, w, target)
        assert torch.equal(fo.linear_cross_entropy(x.t().contiguous().t(), w.t().contiguous().t(), target), same)
        assert torch.equal(fo.linear_cross_entropy(x.reshape(4, 10, 64), w, target.view(4, 10)), same)
        rows = fo.linear_cross_entropy(x.reshape(4, 10, 64), w, target.view(4, 10), reduction="none")
        assert rows.shape == (4, 10) and torch.equal(fo.linear_cross_entropy(x[3], w, target[3], reduction="none"), rows[0, 3])
        assert torch.equal(fo.linear_cross_entropy(x[:1].expand(40, 64), w, target[:1].expand(40), reduction="none"), rows[0, 0].expand(40))


def test_upstream_of_any_stride():
    fo = _fo()
    x, w, target = _inputs(50, 64, 90, BF16)
    each = fo.linear_cross_entropy(x, w, target, reduction="none")
    expanded = torch.autograd.grad(each.sum() * 0.25, (x, w), retain_graph=True)
    spread = torch.full((100,), 0.25, device=DEV)[::2]
    apart = torch.autograd.grad(each, (x, w), spread, retain_graph=True)
    total = torch.autograd.grad(fo.linear_cross_entropy(x, w, target, reduction="sum"), (x, w), torch.tensor(0.25, device=DEV))
    for a, b, c in zip(expanded, apart, total):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_each_gradient_alone():
    fo = _fo()
    for dtype in (F32, BF16, F16):
        x, w, target = _inputs(70, 100, 500, dtype)
        both = torch.autograd.grad(fo.linear_cross_entropy(x, w, target), (x, w))
        assert torch.equal(torch.autograd.grad(fo.linear_cross_entropy(x, w.detach(), target), x)[0], both[0])
        assert torch.equal(torch.autograd.grad(fo.linear_cross_entropy(x.detach(), w, target), w)[0], both[1])


def test_what_stands_in_ignored_rows_does_not_matter():
    fo = _fo()
    for dtype in (F32, BF16, F16):
        x, w, target = _inputs(70, 96, 500, dtype, ignored=0.4)
        target[0] = 3
        want = [fo.linear_cross_entropy(x, w, target, label_smoothing=0.1)]
        want += torch.autograd.grad(want[0], (x, w))
        dirty = x.detach().clone()
        rows = torch.nonzero(target == IGNORE).squeeze(1)
        dirty[rows[0::3]], dirty[rows[1::3]], dirty[rows[2::3]] = float("nan"), float("inf"), torch.finfo(dtype).max
        dirty.requires_grad_()
        got = [fo.linear_cross_entropy(dirty, w, target, label_smoothing=0.1)]
        got += torch.autograd.grad(got[0], (dirty, w))
        assert all(torch.equal(a, b) for a, b in zip(want, got)), dtype
        assert not got[1][rows].any()


@pytest.mark.parametrize("upstream", [float("inf"), float("nan")])
def test_ignored_rows_have_no_gradient_whatever_comes_back(upstream):
    fo = _fo()
    for dtype in (BF16, F16, F32):
        for tokens in (30, 300):
            for reduction in ("mean", "sum"):
                x, w, target = _inputs(tokens, 40, 90, dtype, ignored=0.4)
                loss = fo.linear_cross_entropy(x.requires_grad_(), w.requires_grad_(), target, reduction=reduction)
                dx, _ = torch.autograd.grad(loss, (x, w), torch.full_like(loss, upstream))
                assert (dx[target == IGNORE] == 0).all() and not dx[target != IGNORE].isfinite().any(), (dtype, tokens, reduction)
                loss = fo.linear_cross_entropy(x, w, torch.full_like(target, IGNORE), reduction=reduction)
                dx, dw = torch.autograd.grad(loss, (x, w), torch.full_like(loss, upstream))
                assert (dx == 0).all() and (dw == 0).all(), (dtype, tokens, reduction)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_small_losses_among_large_logits(dtype):
    """One logit of 1000 and 99 of 992, all exact.  exp(-8) is off by 2^-19 of itself (its exponent, 12, by 2^-20), the sum of exponentials, 1.03, by the rounding of fewer than 16 additions
    besides, the logarithm by as much: below 2^-19 in all.  With smoothing the mean of the logits, 992.08, is rounded to 2^-15."""
    fo = _fo()
    x, w = torch.zeros(3, 16, device=DEV, dtype=dtype), torch.zeros(100, 16, device=DEV, dtype=dtype)
    x[:, 0], w[:, 0] = 1.0, 992.0
    target = torch.tensor([0, 41, 99], device=DEV)
    for row, likely in enumerate(target.tolist()):
        weight = w.clone()
        weight[likely, 0] = 1000.0
        for smoothing in (0.0, 0.1):
            want = F.cross_entropy(x.double() @ weight.double().t(), target, label_smoothing=smoothing, reduction="none")
            got = fo.linear_cross_entropy(x, weight, target, label_smoothing=smoothing, reduction="none")
            assert abs(float(got[row]) - float(want[row])) <= 2.0 ** -19 + smoothing * 2.0 ** -14, (row, smoothing)
        # the first value of each row of the matrix's gradient is the logit's: p - 1, where p is off by 2^-19 as well, and rounded to half a step of the type
        weight.requires_grad_()
        fo.linear_cross_entropy(x[row:row + 1], weight, target[row:row + 1]).backward()
        want = torch.softmax(weight.detach().double()[:, 0], 0)
        want[likely] -= 1.0
        off = (weight.grad[:, 0].double() - want).abs()
        assert bool((off <= 2.0 ** -19 * (want.abs() + (want < 0)) + 2 * HALF_STEP[dtype] * want.abs()).all()), (row, off)


def test_all_ignored():
    fo = _fo()
    x, w, target = _inputs(10, 32, 50, BF16)
    target.fill_(7)
    for reduction, want in (("mean", float("nan")), ("sum", 0.0), ("none", 0.0)):
        loss = fo.linear_cross_entropy(x, w, target, ignore_index=7, reduction=reduction)
        assert torch.equal(loss.isnan(), torch.full_like(loss, want).isnan()) and (want != want or not loss.any())
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert not dx.any() and not dw.any()


def test_targets_outside_the_vocabulary():
    fo = _fo()
    x, w, target = _inputs(10, 32, 50, F32)
    good = fo.linear_cross_entropy(x, w, target, reduction="none")
    target[[2, 5, 7]] = torch.tensor([50, -1, (1 << 32) + 1], device=DEV)
    loss = fo.linear_cross_entropy(x, w, target, reduction="none")
    bad = torch.zeros(10, dtype=torch.bool, device=DEV)
    bad[[2, 5, 7]] = True
    assert bool(loss[bad].isnan().all()) and torch.equal(loss[~bad], good[~bad])
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    assert bool(dx[bad].isnan().all()) and bool(dx[~bad].isfinite().all()) and bool(dw.isnan().all())
    assert bool(fo.linear_cross_entropy(x, w, target).isnan())


def test_large_logits():
    """Logits of hundreds: what exp would not hold without the maximum taken off."""
    fo = _fo()
    for dtype in (F32, BF16, F16):
        x, w, target = _inputs(40, 64, 300, dtype)
        x = (x.detach() * 60).requires_grad_()
        loss = fo.linear_cross_entropy(x, w, target, reduction="none")
        want = F.cross_entropy(x.double() @ w.double().t(), target, reduction="none")
        assert bool(loss.isfinite().all()) and bool(((loss.double() - want).abs() <= 2.0 ** -9 + 2.0 ** -14 * want).all())
        assert all(bool(g.isfinite().all()) for g in torch.autograd.grad(loss.sum(), (x, w)))


def test_small_and_large_upstream():
    """What comes in is a power of two times 1: so is what goes out, where the type holds both with all their bits (below its smallest
    normal number it has fewer, so that the products of one rounding are not the other's)."""
    fo = _fo()
    for dtype in (F32, BF16, F16):
        x, w, target = _inputs(40, 64, 300, dtype)
        loss = fo.linear_cross_entropy(x, w, target)
        one = torch.autograd.grad(loss, (x, w), torch.tensor(1.0, device=DEV), retain_graph=True)
        for power in ((-8, 5) if dtype == F16 else (-60, 60)):
            some = torch.autograd.grad(loss, (x, w), torch.tensor(2.0 ** power, device=DEV), retain_graph=True)
            for a, b in zip(one, some):
                held = (a.double() * 2.0 ** power).abs().minimum(a.double().abs()) >= torch.finfo(dtype).tiny
                assert bool((a.double() * 2.0 ** power == b.double())[held].all()), (dtype, power)
        assert not any(g.any() for g in torch.autograd.grad(loss, (x, w), torch.tensor(0.0, device=DEV)))


@pytest.mark.parametrize("divisor", [40, 160])
def test_offsets_beyond_32_bits(divisor):
    fo = _fo()
    width, vocabulary = 4096, 600000       # 2.5e9 values
    w = torch.zeros(vocabulary, width, device=DEV, dtype=BF16)
    rows = torch.tensor([0, 550000, 599999], device=DEV)
    x = torch.randn(3, width, device=DEV).to(BF16)
    w[rows] = (0.3 * x + 0.1 * torch.randn(3, width, device=DEV)).to(BF16) / divisor
    x.requires_grad_(), w.requires_grad_()
    loss = fo.linear_cross_entropy(x, w, rows, reduction="none")
    # the other logits are exactly zero
    x64, w64 = x.detach().double(), w.detach()[rows].double()
    z = x64 @ w64.t()
    lse = (z.exp().sum(1) + (vocabulary - 3)).log()
    e_z = _slack(width, BF16) * (x64.abs() @ w64.abs().t()).amax(1)
    assert bool(((loss.double() - (lse - z.diagonal())).abs() <= 2 * e_z + 2.0 ** -16 + 2.0 ** -22 * loss.double()).all())
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    # What the probabilities are off by is said above.  With 40 they are 1 - 3e-8, and that is all of p - 1: what 1 - p loses to the rounding of fp32 logits
    # of 31 (2^-20 each) is larger than p - 1 itself, so there only the absolute error means something.
    p = (z - lse.unsqueeze(1)).exp()
    g = p - torch.eye(3, device=DEV, dtype=torch.float64)
    off = (2 * e_z + 2.0 ** -16).unsqueeze(1) * p + 2.0 ** -8 * g.abs()
    for got, left, error, right in ((dx, g, off, w64), (dw[rows], g.t(), off.t(), x64)):
        want = left @ right
        bound = error @ right.abs() + _slack(3, BF16) * (left.abs() + error) @ right.abs()
        assert bool(((got.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
    other = (-lse).exp()
    want, bound = other @ x64, (other * (2 * e_z + 2.0 ** -16 + 2.0 ** -8 + 2.0 ** -20)) @ x64.abs()
    for row in (1, 300000, 599998):
        assert bool(((dw[row].double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())


def test_gradient_against_differences():
    fo = _fo()
    x, w, target = _inputs(20, 48, 70, F32, ignored=0.2)
    target[0] = 1
    how = dict(label_smoothing=0.1)
    grads = torch.autograd.grad(fo.linear_cross_entropy(x, w, target, **how), (x, w))
    h = 2.0 ** -5
    with torch.no_grad():
        for k, (leaf, grad) in enumerate(zip((x, w), grads)):
            direction = torch.randn_like(leaf)
            direction /= direction.norm()
            f = lambda step: float(fo.linear_cross_entropy(*[t + (step * direction if i == k else 0.0) for i, t in enumerate((x, w))], target, **how))  # noqa: B023
            slope = (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)
            # fp32 losses of about 3 (2^-22 each, 18 of them over 12 h) and h^4 / 30 of a fifth derivative of order 1
            assert abs(slope - float((grad.double() * direction).sum())) < 18 * 3 * 2.0 ** -22 / (12 * h) + h ** 4 / 30, k


def test_captured_and_replayed():
    fo = _fo()
    x, w, target = (t.detach() for t in _inputs(300, 200, 1000, BF16))

    def both():
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        loss = fo.linear_cross_entropy(*leaves, target, label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for seed in range(3):
        x.copy_(torch.randn(300, 200, generator=torch.Generator().manual_seed(seed)))
        target.copy_(torch.randint(-1, 1000, (300,), generator=torch.Generator().manual_seed(seed)).clamp(min=0))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, both())), seed


def test_refusals():
    fo = _fo()
    x, w, t = torch.zeros(3, 8, device=DEV), torch.zeros(5, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for bad in (dict(x=x.double()), dict(x=x.to(BF16)), dict(x=x[:, :7]), dict(x=x.sum()), dict(x=[0.0]), dict(weight=w[0]), dict(weight=w.cpu()), dict(weight=w.to(F16)),
                dict(target=t[:2]), dict(target=t.float()), dict(target=t.cpu()), dict(target=t.to(torch.uint8)), dict(reduction="max"), dict(label_smoothing=-0.1),
                dict(label_smoothing=1.1), dict(label_smoothing=float("nan")), dict(x=x[:, :0], weight=w[:, :0]), dict(weight=w[:0]), dict(x=x[:0], target=t[:0])):
        with pytest.raises((ValueError, NotImplementedError)):
            fo.linear_cross_entropy(**{**dict(x=x, weight=w, target=t), **bad})
    with pytest.raises(NotImplementedError):
        fo.linear_cross_entropy(x.cpu(), w.cpu(), t.cpu())
    with pytest.raises(RuntimeError, match="too many"):
        fo.linear_cross_entropy(torch.zeros(1, 65537, device=DEV), torch.zeros(2, 65537, device=DEV), t[:1])
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            fo.linear_cross_entropy(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), w, t)
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(fo.linear_cross_entropy(leaf, w + 1.0, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), leaf)

def test_one_derivative_only(host):
    """A second one is refused, also where it is only a part of what is asked for, and whatever came in does not require a gradient."""
    fo = _fo()
    leaf = torch.randn(3, 40, device=DEV, requires_grad=True)
    out = fo.linear_cross_entropy(leaf, torch.randn(9, 40, device=DEV), torch.tensor([1, 2, 8], device=DEV))
    first = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (first.sum() + (leaf * leaf).sum()).backward()
    assert (out.grad_fn.name() == "LinearCrossEntropyBackward") == (host == "nodes")


@pytest.mark.parametrize("upstream", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ignored_rows_of_single_losses_have_no_gradient_whatever_comes_back(dtype, upstream):
    """Losses of single rows that come back with the same infinity: one number for all of them, one for each, one row."""
    fo = _fo()
    for tokens in (1, 30, 300):
        x, w, target = _inputs(tokens, 40, 90, dtype, ignored=0.4)
        for back in (torch.full((), upstream, device=DEV).expand(tokens), torch.full((tokens,), upstream, device=DEV), torch.full((2 * tokens,), upstream, device=DEV)[::2]):
            dx, dw = torch.autograd.grad(fo.linear_cross_entropy(x, w, torch.full_like(target, IGNORE), reduction="none"), (x, w), back)
            assert not dx.any() and not dw.any(), (tokens, back.stride())
            dx, _ = torch.autograd.grad(fo.linear_cross_entropy(x, w, target, reduction="none"), (x, w), back)
            assert not dx[target == IGNORE].any() and not dx[target != IGNORE].isfinite().any(), (tokens, back.stride())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,pieces", [(1, False), (256, False), (257, False), (1000, False), (2100, True)])
def test_what_the_target_loses_is_in_dx_for_any_number_of_rows(tokens, pieces, dtype):
    """p - 1 of every row stands almost in the middle between two numbers of the type, the other words' p next to one, and three quarters of the target's part of dx go up
    against the others'.  Allowed are what the others' p lose, the error of p, 2^-19 as elsewhere here, a contraction over 511 values that are not zero, and one rounding of the result: less than
    0.6 half steps of the target's part in all.  p - 1 rounded as well would be 0.85 to 0.97 more.  The last case has its vocabulary in pieces."""
    fo = _fo()
    half = HALF_STEP[dtype]
    others = 65280 if dtype == BF16 and pieces else 510 if dtype == BF16 else 65504 if pieces else 2047    # powers of two times 1 - 2^-8 and 1 - 2^-11
    g = torch.tensor([2.0 ** -(1 + i % 3) * (1.0 + half * (0.85 + 0.01 * (i % 13))) for i in range(tokens)], dtype=torch.float64)
    logit = torch.log(others * (1 - g) / g)
    x, w = torch.zeros(tokens, 256, dtype=dtype), torch.zeros(others + 1, 256, dtype=dtype)
    x[:, 0] = logit.to(dtype)    # two values, so that their sum has more digits than the type
    x[:, 1] = ((logit - x[:, 0].double()) * 256.0).to(dtype)
    w[0] = torch.randn(256, generator=torch.Generator().manual_seed(tokens)).to(dtype)
    w[1:511] = (0.75 * w[0].float() * others / 510).to(dtype)
    w[:, :2] = 0.0
    w[0, 0], w[0, 1] = 1.0, 2.0 ** -8
    x, w = x.to(DEV), w.to(DEV)
    w64 = w.double()
    p = torch.softmax(x.double() @ w64.t(), 1)
    entry, p = p[:, :1] - 1.0, p[:, 1:2]
    lost, loses = (entry.to(dtype).double() - entry).abs() / entry.abs(), ((32768 * p).to(dtype).double() / 32768 - p).abs()    # of the first, and of each of the others
    assert bool((lost > 0.8 * half).all()) and bool((loses < 0.2 * half * p).all())    # the entries are what they are meant to be
    want = entry * w64[:1] + p * w64[1:511].sum(0)
    error = loses * w64[1:511].abs().sum(0) + 2.0 ** -19 * (w64[:1].abs() + p * w64[1:511].abs().sum(0)) + _slack(511, dtype) * (entry.abs() * w64[:1].abs() + p * w64[1:511].abs().sum(0))
    bound = error + half * (want.abs() + error) + SMALLEST[dtype]
    assert bool((bound < 0.6 * half * entry.abs() * w64[:1].abs() + 2 * SMALLEST[dtype])[:, 2:].all())
    dx = torch.autograd.grad(fo.linear_cross_entropy(x.requires_grad_(), w, torch.zeros(tokens, dtype=torch.int64, device=DEV), reduction="sum"), x)[0]
    far = (dx.double() - want).abs()
    assert bool((far <= bound).all()), float((far / bound).max())
