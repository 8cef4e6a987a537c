"""GPU tests of the MXFP4 quantiser, products and linear layer against the format's definition in 64 bits.

What they allow:
* quantising and dequantising are exact: codes, scale bytes and values equal the definition's;
* a product of two E2M1 values is a multiple of a quarter and at most 36, so a group of 32 sums without rounding; what rounds is the
  fp32 addition of scaled groups.  Over k values that is at most k / 32 additions of at most 2^-23 each (whatever their order
  and whether they round or cut off) of the sum of the magnitudes; the tests allow k 2^-24 + 2^-23 of it, and half a step of
  the type that the result comes in;
* where all groups have one scale and sums stay small, every sum is exact, and so must the result be.
"""

import warnings

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
MOST = {torch.float32: torch.finfo(torch.float32).max, torch.bfloat16: torch.finfo(torch.bfloat16).max, torch.float16: 65504.0}


def _fo():
    import flashoptim_amd

    return flashoptim_amd


def _forms(x):
    """(codes one by one, scale bytes, values) of the rows of `x`, by the definition: search the nearest of eight magnitudes, the
    even code where two are equally near."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    blocks = -(-cols // 128)
    full = torch.zeros(rows, blocks * 128, dtype=torch.float64)
    full[:, :cols] = x
    groups = full.view(rows, blocks * 4, 32)
    finite = groups.isfinite().all(2)
    clean = torch.where(finite.unsqueeze(2), groups, torch.zeros((), dtype=torch.float64))
    largest = clean.abs().amax(2)
    exponent = (torch.frexp(largest)[1] - 1 - 2).clamp(min=-127)
    exponent = torch.where(largest > 0, exponent, -127)
    unit = torch.exp2(exponent.double()).unsqueeze(2)
    size = clean.abs() / unit
    distance = (size.unsqueeze(3) - GRID).abs()
    distance[..., 1::2] += 1e-9     # an even code wins a tie; other distances differ by far more than that, or not at all
    code = distance.argmin(3)
    code = torch.where(size >= 6.0, 7, code)
    values = torch.copysign(GRID[code], clean) * unit
    values = torch.where(finite.unsqueeze(2), values, torch.full((), float("nan"), dtype=torch.float64))
    code = code + 8 * torch.signbit(clean)
    scales = torch.where(finite, exponent + 127, 255).to(torch.uint8)
    return code.view(rows, -1).to(torch.uint8), scales, values.view(rows, -1)[:, :cols]


def _check_form(q, x, what):
    code, scales, _ = _forms(x)
    assert q.shape == tuple(x.shape), what
    assert torch.equal(q.scales.cpu(), scales), (what, "scales")
    got = q.codes.cpu()
    low, high = got & 15, got >> 4
    finite = (scales != 255).repeat_interleave(32, 1)
    want = code
    # where a group is not finite the scale says all; the sign of a zero does not count
    for mine, ref, ok in ((low, want[:, 0::2], finite[:, 0::2]), (high, want[:, 1::2], finite[:, 1::2])):
        same = (mine == ref) | ((mine & 7 == 0) & (ref & 7 == 0)) | ~ok
        assert bool(same.all()), (what, "codes")


def _values(x):
    return _forms(x)[2]


def _random(rows, cols, dtype=torch.float32, seed=0, spread=True):
    """Values whose magnitudes spread over binades within and between rows, ties and zeros among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-4, 5, (rows, cols), generator=g).float())
        x = x * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g).float())
        ties = torch.rand(rows, cols, generator=g) < 0.2
        x = torch.where(ties, torch.round(x * 4) / 4, x)
        x[torch.rand(rows, cols, generator=g) < 0.05] = 0.0
    return x.to(dtype).to(DEV)


def _check_product(got, a, b, what):
    """got against a b' of the values that both stand for (float64, on the CPU or the GPU)."""
    a, b = a.to(DEV), b.to(DEV)
    want, size = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    k = a.shape[1]
    bound = (k * 2.0 ** -24 + 2.0 ** -23) * size
    bound = bound + HALF_STEP[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    held = want.clamp(-MOST[got.dtype], MOST[got.dtype]) if got.dtype != torch.float16 else want
    within = (got.double() - held).abs() <= bound
    if got.dtype == torch.float16:   # beyond its range the type says infinity
        within |= (want.abs() + bound > 65504.0) & got.isinf() & (got.sign() == want.sign())
    assert bool(within.all()), (what, float(((got.double() - want).abs() / bound).max()))


# ------------------------------------------------------------------------------------------------ quantiser


SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 127), (7, 128), (4, 129), (64, 64), (65, 63), (33, 300), (1, 1000), (1000, 1), (129, 257), (250, 1000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forms_along_rows_and_columns(shape, dtype):
    fo = _fo()
    x = _random(*shape, dtype, seed=sum(shape))
    rows, columns = fo.mxfp4_quantize(x), fo.mxfp4_quantize(x, transpose=True)
    _check_form(rows, x, (shape, "rows"))
    _check_form(columns, x.t(), (shape, "columns"))
    for one, both in zip((rows, columns), fo.mxfp4_quantize_both(x)):
        assert torch.equal(one.codes, both.codes) and torch.equal(one.scales, both.scales) and one.shape == both.shape
    for q, values in ((rows, _values(x)), (columns, _values(x.t()))):
        assert torch.equal(q.dequantize(torch.float32).cpu().double(), values)
        assert torch.equal(q.dequantize().cpu().double(), values)
        assert torch.equal(fo.mxfp4_dequantize(q, torch.float16).cpu(), values.to(torch.float16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_binade_and_the_ties_of_each(dtype):
    """A row per binade of the type, subnormal ones among them: its largest value and all values a quarter of a code apart below it."""
    info = torch.finfo(dtype)
    low = {torch.float32: -149, torch.bfloat16: -133, torch.float16: -24}[dtype]
    high = 15 if dtype == torch.float16 else 127
    steps = torch.arange(0, 32, dtype=torch.float64) / 4
    rows = []
    for e in range(low, high + 1):
        row = (steps * 2.0 ** e / 4).clamp(max=float(info.max))
        rows.append(torch.cat([row, -row.flip(0), row * 0.999, torch.full((32,), 2.0 ** e, dtype=torch.float64)]))
    x = torch.stack(rows).to(dtype).to(DEV)
    _check_form(_fo().mxfp4_quantize(x), x, "binades")
    assert torch.equal(_fo().mxfp4_quantize(x).dequantize(torch.float32).cpu().double(), _values(x).float().double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nans_take_their_group_along(dtype):
    fo = _fo()
    x = _random(70, 200, dtype, seed=1)
    x[3, 5], x[40, 64], x[69, 199], x[0, 0] = float("inf"), float("nan"), -float("inf"), float("nan")
    rows, columns = fo.mxfp4_quantize_both(x)
    _check_form(rows, x, "rows")
    _check_form(columns, x.t(), "columns")
    back = rows.dequantize()
    assert torch.equal(back.isnan().cpu(), _values(x).isnan()) and bool(back[3, :32].isnan().all()) and not back[3, 32:].isnan().any()
    y = fo.mxfp4_matmul(rows, fo.mxfp4_quantize(_random(50, 200, seed=2)))
    bad = torch.zeros(70, dtype=torch.bool)
    bad[[0, 3, 40, 69]] = True
    assert torch.equal(y.isnan().all(1).cpu(), bad) and torch.equal(y.isnan().any(1).cpu(), bad)
    few = fo.mxfp4_matmul(x[:5], fo.mxfp4_quantize(_random(50, 200, seed=2)))
    assert torch.equal(few.isnan().all(1).cpu(), bad[:5]) and torch.equal(few.isnan().any(1).cpu(), bad[:5])


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_quantise_like_their_copies(dtype):
    fo = _fo()
    base = _random(140, 309, dtype, seed=3)
    for view in (base[1:, 3:], base[::2, 1:290], base[:, 7:8], base[5:6], base.t(), base[2:130, 9:].t(), base[:, ::3], base[:, :300].expand(140, 300),
                 base[:1, :].expand(50, 309), torch._neg_view(base)):
        for got, want in zip(fo.mxfp4_quantize_both(view), fo.mxfp4_quantize_both(view.clone(memory_format=torch.contiguous_format))):
            assert got.shape == want.shape and torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0)])
def test_matrices_without_elements(shape):
    fo = _fo()
    x = torch.empty(shape, device=DEV)
    rows, columns = fo.mxfp4_quantize_both(x)
    assert rows.shape == shape and columns.shape == shape[::-1]
    assert rows.dequantize().shape == shape


def test_more_elements_than_32_bits_count():
    fo = _fo()
    rows, cols = 70000, 33000
    assert rows * cols > 2 ** 31
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    part = _random(300, 200, torch.bfloat16, seed=4)
    x[-300:, -200:] = part
    x[:300, :200] = part
    by_row, by_column = fo.mxfp4_quantize_both(x)
    assert torch.equal(by_row.dequantize()[:300, :200].cpu().double(), _values(part))
    assert torch.equal(by_column.dequantize()[:200, :300].cpu().double(), _values(part.t()))
    lead = cols - 200 - (cols - 200) // 32 * 32
    want = torch.zeros(300, lead + 200, device=DEV, dtype=torch.bfloat16)
    want[:, lead:] = part
    assert torch.equal(by_row.dequantize()[-300:, -200 - lead:].cpu().double(), _values(want))
    lead = rows - 300 - (rows - 300) // 32 * 32
    want = torch.zeros(200, lead + 300, device=DEV, dtype=torch.bfloat16)
    want[:, lead:] = part.t()
    assert torch.equal(by_column.dequantize()[-200:, -300 - lead:].cpu().double(), _values(want))


# ------------------------------------------------------------------------------------------------ products


PRODUCTS = [(1, 1, 1), (1, 5, 31), (2, 33, 32), (7, 16, 129), (16, 250, 1000), (17, 64, 256), (33, 100, 384), (64, 128, 640), (65, 65, 65),
            (128, 256, 128), (130, 257, 1000), (300, 70, 2730), (513, 500, 250), (1003, 1000, 513), (1024, 1536, 2048)]


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_product_against_float64(shape, out):
    fo = _fo()
    m, n, k = shape
    a, b = _random(m, k, seed=m), _random(n, k, seed=n + 1)
    qa, qb = fo.mxfp4_quantize(a), fo.mxfp4_quantize(b)
    va, vb = _values(a), _values(b)
    _check_product(fo.mxfp4_matmul(qa, qb, out), va, vb, (shape, out))
    for dtype in DTYPES:      # a plain first operand, of every type
        x = a.to(dtype)
        _check_product(fo.mxfp4_matmul(x, qb, out), _values(x), vb, (shape, out, dtype))


@pytest.mark.parametrize("shape", PRODUCTS)
def test_sums_that_fit_are_exact(shape):
    """Grid values of one scale: sums are multiples of a quarter below 2^20."""
    fo = _fo()
    m, n, k = shape
    g = torch.Generator().manual_seed(k)
    a, b = (GRID[torch.randint(0, 8, (r, k), generator=g)] * (2.0 * torch.randint(0, 2, (r, k), generator=g) - 1.0) for r in (m, n))
    a[:, ::32], b[:, ::32] = 6.0, -4.0     # every group has the scale 1
    want = a @ b.t()
    qa, qb = fo.mxfp4_quantize(a.float().to(DEV)), fo.mxfp4_quantize(b.float().to(DEV))
    assert torch.equal(fo.mxfp4_matmul(qa, qb, torch.float32).cpu().double(), want)
    assert torch.equal(fo.mxfp4_matmul(a.to(torch.bfloat16).to(DEV), qb, torch.float32).cpu().double(), want)


@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65])
@pytest.mark.parametrize("n,k", [(250, 1000), (4096, 128), (31, 14336), (130, 33)])
def test_few_tokens_equal_the_product_of_forms(tokens, n, k):
    """However many rows there are, and whoever quantises them."""
    fo = _fo()
    x, w = _random(tokens, k, torch.bfloat16, seed=tokens), _random(n, k, seed=n)
    qw = fo.mxfp4_quantize(w)
    _check_product(fo.mxfp4_linear(x, qw), _values(x), _values(w), (tokens, n, k))
    wide = _random(tokens, k + 5, torch.bfloat16, seed=tokens)
    assert torch.equal(fo.mxfp4_linear(wide[:, 3:3 + k], qw), fo.mxfp4_linear(wide[:, 3:3 + k].contiguous(), qw))
    turned = x.t().contiguous().t()
    assert torch.equal(fo.mxfp4_linear(turned, qw), fo.mxfp4_linear(x, qw))


def test_extreme_scales_meet():
    """Rows near the ends of fp32's range: the product's scale is the sum of both exponents."""
    fo = _fo()
    g = torch.Generator().manual_seed(5)
    for ea, eb in ((-100, 100), (60, 60), (-60, -60), (120, -120), (-126, 124)):
        for m in (3, 100):
            a, b = torch.randn(m, 200, generator=g).to(DEV) * 2.0 ** ea, torch.randn(40, 200, generator=g).to(DEV) * 2.0 ** eb
            got = fo.mxfp4_matmul(fo.mxfp4_quantize(a), fo.mxfp4_quantize(b), torch.float32)
            _check_product(got, _values(a), _values(b), (ea, eb, m))
            _check_product(fo.mxfp4_matmul(a, fo.mxfp4_quantize(b), torch.float32), _values(a), _values(b), (ea, eb, m, "plain"))


@pytest.mark.parametrize("m,n,k", [(0, 5, 7), (5, 0, 7), (5, 7, 0), (0, 0, 0)])
def test_products_without_elements(m, n, k):
    fo = _fo()
    a, b = torch.ones(m, k, device=DEV), torch.ones(n, k, device=DEV)
    for left in (a, fo.mxfp4_quantize(a)):
        got = fo.mxfp4_matmul(left, fo.mxfp4_quantize(b))
        assert got.shape == (m, n) and not got.any()


# ------------------------------------------------------------------------------------------------ the layer


def _linear_reference(x, w, dy):
    x, w, dy = (t.detach().cpu() for t in (x, w, dy))
    return ((_values(x), _values(w)), (_values(dy), _values(w.t())), (_values(dy.t()), _values(x.t())))


LAYERS = [(1, 1, 1), (3, 33, 5), (64, 128, 96), (65, 100, 130), (1, 1000, 250), (250, 1, 64), (130, 250, 1), (512, 256, 384), (1003, 500, 257)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,inner,outer", LAYERS)
def test_layer_and_its_gradients(tokens, inner, outer, dtype):
    fo = _fo()
    x = _random(tokens, inner, dtype, seed=1).requires_grad_()
    w = _random(outer, inner, dtype, seed=2, spread=False).requires_grad_()
    dy = _random(tokens, outer, dtype, seed=3)
    y = fo.mxfp4_linear(x, w)
    assert y.dtype == dtype and y.shape == (tokens, outer)
    y.backward(dy)
    for got, (a, b), what in zip((y.detach(), x.grad, w.grad), _linear_reference(x, w, dy), ("y", "dx", "dw")):
        assert got.dtype == dtype
        _check_product(got, a, b, (what, tokens, inner, outer))


def _grid_matrix(rows, cols, seed):
    """Grid values of which rows and columns alike have the scale 1 in every group: both forms hold them exactly."""
    g = torch.Generator().manual_seed(seed)
    x = GRID[torch.randint(0, 8, (rows, cols), generator=g)] * (2.0 * torch.randint(0, 2, (rows, cols), generator=g) - 1.0)
    x[:, ::32], x[::32, :] = 4.0, -6.0
    return x.float().to(DEV)


def test_gradients_against_differences():
    """On values that both forms hold the layer is linear, so differences are the gradient, exactly: loss(x + step) - loss(x) for a
    step from one grid value to another, at every 7th place of x and of the weight."""
    fo = _fo()
    tokens, inner, outer = 40, 70, 50
    x, w, dy = _grid_matrix(tokens, inner, 1), _grid_matrix(outer, inner, 2), _grid_matrix(tokens, outer, 3)

    def loss(x, w):
        return (fo.mxfp4_linear(x, w).double() * dy.double()).sum().item()

    leaf, weight = x.clone().requires_grad_(), w.clone().requires_grad_()
    fo.mxfp4_linear(leaf, weight).backward(dy)
    base = loss(x, w)
    for tensor, grad, call in ((x, leaf.grad, lambda t: loss(t, w)), (w, weight.grad, lambda t: loss(x, t))):
        for at in range(0, tensor.numel(), 7):
            i, j = divmod(at, tensor.shape[1])
            if i % 32 == 0 or j % 32 == 0:
                continue    # these keep the scales
            moved = tensor.clone()
            moved[i, j] = 2.0 if tensor[i, j] != 2.0 else -1.0
            assert call(moved) - base == (moved[i, j] - tensor[i, j]).item() * grad[i, j].item(), at


def test_gradients_of_some_inputs_only():
    fo = _fo()
    x, w, dy = _random(50, 70, torch.bfloat16, seed=1), _random(30, 70, torch.bfloat16, seed=2), _random(50, 30, torch.bfloat16, seed=3)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    fo.mxfp4_linear(a, b).backward(dy)
    c = x.clone().requires_grad_()
    fo.mxfp4_linear(c, w).backward(dy)
    d = w.clone().requires_grad_()
    fo.mxfp4_linear(x, d).backward(dy)
    assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)
    with torch.no_grad():
        assert torch.equal(fo.mxfp4_linear(a, b), fo.mxfp4_linear(x, w))
    mixed = fo.mxfp4_linear(x, w.float().requires_grad_())
    assert torch.equal(mixed, fo.mxfp4_linear(x, w)) and mixed.dtype == torch.bfloat16


def test_shared_and_broadcast_operands_add_their_gradients():
    fo = _fo()
    w = _random(30, 70, seed=2).requires_grad_()
    x, dy = _random(50, 70, seed=1), _random(50, 30, seed=3)
    (fo.mxfp4_linear(x, w) + fo.mxfp4_linear(x, w)).backward(dy)
    single = w.detach().clone().requires_grad_()
    fo.mxfp4_linear(x, single).backward(dy)
    assert torch.equal(w.grad, 2.0 * single.grad)
    row = _random(1, 70, seed=4).requires_grad_()
    fo.mxfp4_linear(row.expand(50, 70), w).backward(dy)
    whole = row.detach().expand(50, 70).contiguous().requires_grad_()
    fo.mxfp4_linear(whole, w).backward(dy)
    assert torch.allclose(row.grad, whole.grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-5 * float(whole.grad.abs().sum(0).max()))


def test_gradients_that_come_with_strides():
    """Sums hand down expanded gradients, transposes transposed ones."""
    fo = _fo()
    w, x = _random(30, 70, seed=2), _random(50, 70, seed=1)
    for spread in (lambda y: y.sum(), lambda y: y.t().contiguous().sum(1).sum(), lambda y: y[::2, 3:].sum(), lambda y: (y.t() @ _random(50, 5, seed=6)).sum()):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = fo.mxfp4_linear(a, b)
        spread(y).backward()
        z = y.detach().clone().requires_grad_()
        spread(z).backward()
        c, d = x.clone().requires_grad_(), w.clone().requires_grad_()
        fo.mxfp4_linear(c, d).backward(z.grad.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)


def test_layer_takes_any_leading_shape_and_module_adds_its_bias():
    fo = _fo()
    torch.manual_seed(0)
    layer = fo.MXFP4Linear(70, 30).to(DEV).to(torch.bfloat16)
    x = _random(24, 70, torch.bfloat16, seed=1)
    flat = layer(x)
    assert torch.equal(flat, fo.mxfp4_linear(x, layer.weight) + layer.bias)
    assert torch.equal(layer(x.view(2, 3, 4, 70)), flat.view(2, 3, 4, 30))
    assert torch.equal(layer(x[0]), layer(x[:1])[0])
    held = fo.mxfp4_quantize(layer.weight)
    assert torch.equal(fo.mxfp4_linear(x.view(2, 12, 70), held), fo.mxfp4_linear(x, held).view(2, 12, 30))
    flat.float().sum().backward()
    assert layer.weight.grad is not None and torch.equal(layer.bias.grad, torch.full_like(layer.bias, 24.0))


@pytest.mark.parametrize("tokens,inner,outer", LAYERS)
def test_training_and_serving_agree(tokens, inner, outer):
    """The layer's output with the weight as a parameter and held in MXFP4."""
    fo = _fo()
    x, w = _random(tokens, inner, torch.bfloat16, seed=1), _random(outer, inner, torch.bfloat16, seed=2)
    held = fo.mxfp4_quantize(w)
    _check_product(fo.mxfp4_linear(x, held), _values(x), _values(w), "serving")
    leaf = x.clone().requires_grad_()
    y = fo.mxfp4_linear(leaf, held)
    dy = _random(tokens, outer, torch.bfloat16, seed=3)
    y.backward(dy)
    # the frozen weight's values, with their scales along the other axis
    _check_product(leaf.grad, _values(dy), _values(_values(w).t()), "frozen gradient")


def test_on_another_stream():
    fo = _fo()
    x, w, dy = _random(300, 250, torch.bfloat16, seed=1), _random(200, 250, torch.bfloat16, seed=2), _random(300, 200, torch.bfloat16, seed=3)

    def step():
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = fo.mxfp4_linear(a, b)
        return (y, *torch.autograd.grad(y, (a, b), dy), fo.mxfp4_linear(x[:7], fo.mxfp4_quantize(w)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = [step() for _ in range(3)]
    side.synchronize()
    for each in got:
        for a, b in zip(each, want):
            assert torch.equal(a, b)


def test_in_a_graph():
    fo = _fo()
    w = _random(200, 250, torch.bfloat16, seed=2)
    held = fo.mxfp4_quantize(w)
    few, many = _random(5, 250, torch.bfloat16, seed=1), _random(300, 250, torch.bfloat16, seed=1)

    def run():
        return fo.mxfp4_linear(few, held), fo.mxfp4_linear(many, w), fo.mxfp4_dequantize(fo.mxfp4_quantize(many, transpose=True))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(3):
        few.copy_(_random(5, 250, torch.bfloat16, seed=10 + seed))
        many.copy_(_random(300, 250, torch.bfloat16, seed=20 + seed))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_a_network_trains_in_it():
    """Two MXFP4 layers, their matrices under FlashMuon and the rest under FlashAdamW, fit a random network's outputs: the loss falls to a
    fifth (what the 4-bit products leave of it)."""
    fo = _fo()
    torch.manual_seed(1)
    teacher = nn.Sequential(nn.Linear(64, 128), nn.GELU(), nn.Linear(128, 32)).to(DEV)
    student = nn.Sequential(fo.MXFP4Linear(64, 256), nn.GELU(), fo.MXFP4Linear(256, 32)).to(DEV).to(torch.bfloat16)
    matrices = [p for p in student.parameters() if p.dim() == 2]
    rest = [p for p in student.parameters() if p.dim() != 2]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        opts = [fo.FlashMuon(matrices, lr=0.02, weight_decay=0.0), fo.FlashAdamW(rest, lr=1e-2, weight_decay=0.0)]
    losses = []
    for step in range(300):
        x = torch.randn(512, 64, device=DEV)
        with torch.no_grad():
            want = teacher(x)
        for opt in opts:
            opt.param_groups[0]["lr"] = opt.defaults["lr"] * (1.0 - step / 300)
            opt.zero_grad()
        loss = (student(x.to(torch.bfloat16)).float() - want).square().mean()
        loss.backward()
        for opt in opts:
            opt.step()
        losses.append(loss.item())
    assert sum(losses[-10:]) < 0.2 * sum(losses[:3]) / 3 * 10, (losses[0], losses[-1])


def test_the_example_trains_and_answers():
    from examples.mxfp4_muon import main

    result = main(["--steps", "400"])
    assert result["last"] < result["entropy"] + 0.3 and result["allowed"] > 0.95


# ------------------------------------------------------------------------------------------------ refusals


def test_refusals():
    fo = _fo()
    x = torch.zeros(4, 40, device=DEV)
    q = fo.mxfp4_quantize(x)
    for call in (fo.mxfp4_quantize, fo.mxfp4_quantize_both):
        with pytest.raises(NotImplementedError):
            call(x.cpu())
        for bad in (x.double(), x.int(), x[0], x.view(2, 2, 40)):
            with pytest.raises(ValueError):
                call(bad)
    with pytest.raises(ValueError):
        fo.mxfp4_dequantize(x)
    with pytest.raises(ValueError):
        fo.mxfp4_dequantize(q, torch.float64)
    with pytest.raises(NotImplementedError):
        fo.mxfp4_dequantize(q.to("cpu"))
    with pytest.raises(ValueError):
        fo.mxfp4_matmul(q, x)
    with pytest.raises(ValueError):
        fo.mxfp4_matmul(q, q, torch.int32)
    with pytest.raises(ValueError, match="contract"):
        fo.mxfp4_matmul(q, fo.mxfp4_quantize(torch.zeros(4, 41, device=DEV)))
    with pytest.raises(ValueError):
        fo.mxfp4_matmul(q.to("cpu"), q)
    with pytest.raises(ValueError, match="fit"):
        fo.mxfp4_linear(x, torch.zeros(5, 41, device=DEV))
    with pytest.raises(ValueError, match="fit"):
        fo.mxfp4_linear(torch.zeros((), device=DEV), q)
    with pytest.raises(ValueError):
        fo.mxfp4_linear(x, torch.zeros(5, 40))
    with pytest.raises(ValueError):
        fo.mxfp4_linear(x, torch.zeros(2, 5, 40, device=DEV))
    with pytest.raises(ValueError):
        fo.mxfp4_linear(x.double(), q)
    with pytest.raises(ValueError):
        fo.mxfp4_linear(x, torch.zeros(5, 40, device=DEV, dtype=torch.float64))
    for codes, scales, shape in ((q.codes[:, :32], q.scales, (4, 40)), (q.codes, q.scales[:3], (4, 40)), (q.codes, q.scales, (4, 200)),
                                 (q.codes.float(), q.scales, (4, 40)), (q.codes, q.scales.int(), (4, 40)), (q.codes, q.scales.cpu(), (4, 40)),
                                 (torch.zeros(64, 4, dtype=torch.uint8, device=DEV).t(), q.scales, (4, 40)), (q.codes, q.scales, (-1, 40))):
        with pytest.raises(ValueError):
            fo.MXFP4Tensor(codes, scales, shape)
