"""GPU tests of the residual's addition with the root-mean-square norm, its gradients and its MXFP4 form, against 64 bits.

What they allow, with u = 2^-24:
* the stream is one fp32 addition and one rounding, as in torch: exact;
* the mean of squares is summed in fp64, so u of it for its rounding and u for the eps, half of both in its root; that is off by a unit (2 u), and the two
  products by u each: 5 u, and half a step of the type; 2^-19 is allowed;
* in the gradient the mean of dn n, where a value passes at most 32 + 14 additions, is off by at most 46 u of the mean of the magnitudes besides; a term has 2^-18 of its magnitude, the result
  half a step;
* a sum over rows is made of at most 1 + rows / 512 + 72 additions: that many u of the magnitudes' sum, and 2^-19 for n.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SMALLEST = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}
WIDTHS = [1, 7, 8, 31, 128, 250, 512, 513, 2048, 2730, 4096, 4100, 8192, 8200, 16379, 16384]


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


def _close(got, want, slack, what):
    """got within `slack` of `want` before it was rounded to its type."""
    bound = slack + HALF_STEP[got.dtype] * (want.abs() + slack) + SMALLEST[got.dtype]
    far = (got.double() - want).abs()
    assert bool((far <= bound).all()), (what, float((far / bound).max()))


def _exact(s, w, eps, dy=None, dstream=None):
    """y, and with dy the gradients and the magnitudes of their terms, of the stream s."""
    s, w = s.double(), 1.0 if w is None else w.double()
    inverse = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    n = s * inverse
    out = [n * w]
    if dy is not None:
        dy = dy.double()
        dn = dy * w
        ds = inverse * (dn - n * (dn * n).mean(1, keepdim=True))
        size = inverse * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True))
        if dstream is not None:
            ds, size = ds + dstream.double(), size + dstream.double().abs()
        out += [ds, size, (dy * n).sum(0), (dy * n).abs().sum(0)]
    return out


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_and_gradients(width, types):
    fo = _fo()
    dtype, stream_dtype = types
    g = torch.Generator(device=DEV).manual_seed(width)
    for rows, with_residual, w_dtype in ((1, True, dtype), (5, False, F32), (67, True, BF16), (1100 if width < 1000 else 3, True, None)):
        what = (width, types, rows, with_residual, w_dtype)
        randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: B023
        x = (randn(rows, width) * torch.exp2(torch.randint(-6, 6, (rows, 1), generator=g, device=DEV).float())).to(dtype).requires_grad_()
        residual = randn(rows, width).to(stream_dtype).requires_grad_() if with_residual else None
        w = None if w_dtype is None else (1.0 + 0.3 * randn(width)).to(w_dtype).requires_grad_()
        dy, dstream = randn(rows, width).to(dtype), randn(rows, width).to(stream_dtype) if with_residual else None
        got = fo.rms_norm(x, w, residual, eps=1e-5)
        if with_residual:
            y, s = got
            assert torch.equal(s, (x.detach().float() + residual.detach().float()).to(stream_dtype)), what
        else:
            y, s = got, x
        want_y, want_ds, size, want_dw, dw_size = _exact(s.detach(), None if w is None else w.detach(), 1e-5, dy, dstream)
        _close(y.detach(), want_y, 2.0 ** -19 * want_y.abs(), (what, "y"))
        leaves = [t for t in (x, residual, w) if t is not None]
        outputs, upstream = ((y, s), (dy, dstream)) if with_residual else ((y,), (dy,))
        grads = torch.autograd.grad(outputs, leaves, upstream, retain_graph=True)
        for leaf, grad in zip(leaves, grads):
            assert grad.dtype == leaf.dtype and grad.shape == leaf.shape, what
            if leaf is w:
                _close(grad, want_dw, (2.0 ** -19 + (73 + rows / 512) * 2.0 ** -24) * dw_size, (what, "dw"))
            else:
                _close(grad, want_ds, 2.0 ** -18 * size, (what, "dx"))
        for a, b in zip(grads, torch.autograd.grad(outputs, leaves, upstream)):
            assert torch.equal(a, b), what
        with torch.no_grad():
            plain = fo.rms_norm(x, w, residual, eps=1e-5)
            assert torch.equal(plain[0], y) and torch.equal(plain[1], s) if with_residual else torch.equal(plain, y), what


@pytest.mark.parametrize("width", [1, 31, 33, 128, 129, 250, 512, 520, 2730, 4096, 5000, 16300])
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_mxfp4_output_is_the_quantised_norm(width, types):
    """Bit for bit what the quantiser makes of the norm in fp32 of the same stream."""
    fo = _fo()
    dtype, stream_dtype = types
    for rows in (1, 9):
        x = (3.0 * torch.randn(rows, width, device=DEV)).to(dtype)
        residual = torch.randn(rows, width, device=DEV).to(stream_dtype)
        w = (1.0 + 0.3 * torch.randn(width, device=DEV)).to(dtype)
        if rows > 1:
            x[3], residual[3] = 0.0, 0.0
            x[4, 0] = float("nan")
        q, s = fo.rms_norm_mxfp4(x, w, residual, eps=1e-5)
        want = fo.mxfp4_quantize(fo.rms_norm(s.float(), w, eps=1e-5))
        assert torch.equal(s, (x.float() + residual.float()).to(stream_dtype)) or rows > 1
        assert q.shape == want.shape and torch.equal(q.scales, want.scales) and torch.equal(q.codes, want.codes), (width, types, rows)
        only = fo.rms_norm_mxfp4(x, None)
        want = fo.mxfp4_quantize(fo.rms_norm(x.float(), eps=1e-6))
        assert torch.equal(only.scales, want.scales) and torch.equal(only.codes, want.codes), (width, types, rows)


def test_mxfp4_output_goes_into_the_products():
    fo = _fo()
    x, r = torch.randn(5, 256, device=DEV).to(BF16), torch.randn(5, 256, device=DEV).to(BF16)
    w, layer = torch.ones(256, device=DEV, dtype=BF16), fo.mxfp4_quantize(torch.randn(300, 256, device=DEV))
    q, s = fo.rms_norm_mxfp4(x, w, r)
    same = fo.mxfp4_quantize(q.dequantize(F32))
    assert torch.equal(same.codes, q.codes) and torch.equal(same.scales, q.scales)
    assert torch.equal(fo.mxfp4_matmul(q, layer), fo.mxfp4_matmul(same, layer))


def test_rows_of_extreme_values():
    """fp32 does not hold these rows' squares; rows of zeros have the inverse root of eps."""
    fo = _fo()
    for size in (1e30, 3e37, 1e-25, 1e-30):
        s = torch.randn(4, 600, device=DEV) * size
        s = s.requires_grad_()
        dy = torch.randn(4, 600, device=DEV)
        y = fo.rms_norm(s, eps=0.0)
        want, ds, magnitude, _, _ = _exact(s.detach(), None, 0.0, dy)
        _close(y.detach(), want, 2.0 ** -19 * want.abs(), size)
        _close(torch.autograd.grad(y, s, dy)[0], ds, 2.0 ** -18 * magnitude, size)
    zeros = torch.zeros(3, 40, device=DEV, requires_grad=True)
    y = fo.rms_norm(zeros, eps=1e-6)
    assert not y.any() and bool((torch.autograd.grad(y.sum(), zeros)[0] - 1e3).abs().max() < 0.01)


def test_infinities_and_nan_stay_in_their_rows():
    fo = _fo()
    x = torch.randn(6, 300, device=DEV)
    clean = fo.rms_norm(x)
    x[1, 5], x[3, 299] = float("inf"), float("nan")
    y = fo.rms_norm(x)
    rows = torch.tensor([0, 2, 4, 5], device=DEV)
    assert torch.equal(y[rows], clean[rows]) and bool(y[3].isnan().all()) and bool(y[1, 5].isnan())


def test_shapes_and_strides():
    fo = _fo()
    wide = torch.randn(4, 5, 90, device=DEV).to(BF16)
    x, residual, w = wide[:, :, 3:73], torch.randn(4, 5, 100, device=DEV).to(BF16)[:, :, ::1][:, :, 20:90], torch.randn(140, device=DEV)[::2]
    y, s = fo.rms_norm(x, w, residual)
    want_y, want_s = fo.rms_norm(x.contiguous(), w.contiguous(), residual.contiguous())
    assert y.shape == x.shape and torch.equal(y, want_y) and torch.equal(s, want_s)
    flat = wide[0, :, 3:73]
    assert torch.equal(fo.rms_norm(flat), fo.rms_norm(flat.contiguous()))
    assert torch.equal(fo.rms_norm(flat.t()), fo.rms_norm(flat.t().contiguous()))
    assert torch.equal(fo.rms_norm(flat[0]), fo.rms_norm(flat)[0])
    assert torch.equal(fo.rms_norm(flat[:1].expand(7, 70)), fo.rms_norm(flat[:1]).expand(7, 70))
    assert fo.rms_norm(flat[:0]).shape == (0, 70)
    # the gradients' own strides
    leaf = flat.detach().clone().requires_grad_()
    for dy in (torch.randn(70, 5, device=DEV).to(BF16).t(), torch.randn(1, 70, device=DEV).to(BF16).expand(5, 70), torch.randn(5, 99, device=DEV).to(BF16)[:, 7:77]):
        assert torch.equal(torch.autograd.grad(fo.rms_norm(leaf), leaf, dy)[0], torch.autograd.grad(fo.rms_norm(leaf), leaf, dy.contiguous())[0])
    # no rows
    none, w = torch.zeros(0, 70, device=DEV, requires_grad=True), torch.ones(70, device=DEV, requires_grad=True)
    dx, dw = torch.autograd.grad(fo.rms_norm(none, w).sum(), (none, w))
    assert dx.shape == (0, 70) and dw.shape == (70,) and not dw.any()


def test_each_gradient_alone():
    fo = _fo()
    for dtype, stream_dtype in TYPES:
        x, r = torch.randn(9, 77, device=DEV).to(dtype), torch.randn(9, 77, device=DEV).to(stream_dtype)
        w, dy, ds = torch.randn(77, device=DEV).to(dtype), torch.randn(9, 77, device=DEV).to(dtype), torch.randn(9, 77, device=DEV).to(stream_dtype)
        leaves = [t.clone().requires_grad_() for t in (x, w, r)]
        every = torch.autograd.grad(fo.rms_norm(*leaves), leaves, (dy, ds))
        for k in range(3):
            some = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, r))]
            assert torch.equal(torch.autograd.grad(fo.rms_norm(*some), some[k], (dy, ds))[0], every[k]), (dtype, stream_dtype, k)
        # only one of the two outputs goes on
        y, s = fo.rms_norm(*leaves)
        from_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        zero = torch.autograd.grad((y, s), leaves, (dy, torch.zeros_like(ds)), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(from_y, zero))
        dx, dr = torch.autograd.grad(s, (leaves[0], leaves[2]), ds)
        assert torch.equal(dx, ds.to(dtype)) and torch.equal(dr, ds)


def test_a_stream_changed_in_place_is_noticed():
    fo = _fo()
    x, r = torch.randn(4, 30, device=DEV, requires_grad=True), torch.randn(4, 30, device=DEV)
    y, s = fo.rms_norm(x, None, r)
    s.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_gradient_against_differences():
    fo = _fo()
    x, r, w = (torch.randn(3, 50, device=DEV, requires_grad=True), torch.randn(3, 50, device=DEV, requires_grad=True), torch.randn(50, device=DEV, requires_grad=True))
    dy, ds = torch.randn(3, 50, device=DEV), torch.randn(3, 50, device=DEV)
    grads = torch.autograd.grad(fo.rms_norm(x, w, r), (x, w, r), (dy, ds))
    h = 2.0 ** -7

    def at(k, direction, step):
        args = [t.detach() + (step * direction if i == k else 0.0) for i, t in enumerate((x, w, r))]
        y, s = fo.rms_norm(*args)
        return float((y.double() * dy).sum() + (s.double() * ds).sum())

    for k, (leaf, grad) in enumerate(zip((x, w, r), grads)):
        direction = torch.randn_like(leaf)
        slope = (8 * (at(k, direction, h) - at(k, direction, -h)) - (at(k, direction, 2 * h) - at(k, direction, -2 * h))) / (12 * h)
        # fourth differences: h^4 / 30 of the fifth derivative (1e-7 here), and fp32's 150 roundings of order 1 over h
        assert abs(slope - float((grad.double() * direction).sum())) < 5e-3, k


def test_captured_and_replayed():
    fo = _fo()
    x, r, w = torch.randn(300, 1000, device=DEV).to(BF16), torch.randn(300, 1000, device=DEV).to(BF16), torch.randn(1000, device=DEV).to(BF16)

    def both():
        leaves = [t.detach().requires_grad_() for t in (x, w, r)]
        y, s = fo.rms_norm(*leaves)
        q, _ = fo.rms_norm_mxfp4(x, w, r)
        return [y.detach(), s.detach(), q.codes, q.scales, *torch.autograd.grad((y, s), leaves, (r, x))]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for seed in range(3):
        x.copy_(torch.randn(300, 1000, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, both())), seed


def test_module():
    fo = _fo()
    layer = fo.FlashRMSNorm(64, eps=1e-5, device=DEV, dtype=BF16)
    x, r = torch.randn(2, 3, 64, device=DEV).to(BF16), torch.randn(2, 3, 64, device=DEV).to(BF16)
    y, s = layer(x, r)
    assert torch.equal(layer(s), y) and list(layer.state_dict()) == ["weight"]
    y.sum().backward()
    assert layer.weight.grad.shape == (64,)
    assert fo.FlashRMSNorm(64, elementwise_affine=False)(x).shape == x.shape


def test_refusals():
    fo = _fo()
    x = torch.zeros(4, 40, device=DEV)
    for call in (fo.rms_norm, fo.rms_norm_mxfp4):
        for bad in (dict(x=x.double()), dict(x=x.int()), dict(x=[1.0]), dict(x=torch.zeros((), device=DEV)), dict(weight=x[0, :39]), dict(weight=x), dict(weight=x[0].cpu()),
                    dict(weight=x[0].double()), dict(residual=x[:3]), dict(residual=x.to(BF16)), dict(residual=x.cpu()), dict(residual=x.double()), dict(eps=-1.0),
                    dict(eps=float("nan")), dict(eps=float("inf"))):
            with pytest.raises((ValueError, NotImplementedError)):
                call(**{**dict(x=x), **bad})
        with pytest.raises(NotImplementedError):
            call(x.cpu())
        with pytest.raises(RuntimeError, match="too long"):
            call(torch.zeros(1, 16385, device=DEV))
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(ValueError):
        fo.rms_norm_mxfp4(x.view(2, 2, 40))
    with pytest.raises(ValueError):
        fo.rms_norm(x.to(BF16), residual=x.to(F16))
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(fo.rms_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), leaf)

def test_one_derivative_only(host):
    """A second one is refused, also where it is only a part of what is asked for, and whatever came in does not require a gradient."""
    fo = _fo()
    leaf, w = torch.randn(3, 40, device=DEV, requires_grad=True), torch.ones(40, device=DEV)
    out = fo.rms_norm(leaf, w)
    first = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (first.sum() + (leaf * leaf).sum()).backward()
    assert (out.grad_fn.name() == "RMSNormBackward") == (host == "nodes")


def test_a_stream_alone_brings_its_gradient_alone():
    """Where the norm's output is not used, what stands in its rows does not reach the gradients: infinities, NaN, rows of zeros without eps."""
    fo = _fo()
    for dtype, stream_dtype in TYPES:
        x, r = torch.randn(6, 77, device=DEV).to(dtype), torch.randn(6, 77, device=DEV).to(stream_dtype)
        w, ds = torch.randn(77, device=DEV).to(dtype), torch.randn(6, 77, device=DEV).to(stream_dtype)
        x[1, 3], r[2, 70], x[4], r[4] = float("inf"), float("nan"), 0.0, 0.0
        for shape in ((6, 77), (2, 3, 77)):
            for eps in (0.0, 1e-6):
                leaves = [x.clone().view(shape).requires_grad_(), w.clone().requires_grad_(), r.clone().view(shape).requires_grad_()]
                y, s = fo.rms_norm(*leaves, eps=eps)
                dx, dw, dr = torch.autograd.grad(s, leaves, ds.view(shape))
                assert torch.equal(dx, ds.view(shape).to(dtype)) and torch.equal(dr, ds.view(shape)) and dw.shape == w.shape and dw.dtype == dtype and not dw.any()
                for k in (0, 2):
                    some = [t.detach().clone().requires_grad_(i == k) for i, t in enumerate(leaves)]
                    s = fo.rms_norm(*some, eps=eps)[1]
                    assert torch.equal(torch.autograd.grad(s, some[k], ds.view(shape))[0], dx if k == 0 else dr)
    leaves = [torch.randn(6, 77, device=DEV, requires_grad=True) for _ in range(2)]
    s = fo.rms_norm(leaves[0], None, leaves[1])[1]
    s.sum().backward()
    assert leaves[0].grad.data_ptr() != leaves[1].grad.data_ptr()
    s = fo.rms_norm(leaves[0], None, leaves[1])[1]
    (first,) = torch.autograd.grad(s, leaves[0], torch.ones_like(s), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        first.sum().backward()


@pytest.mark.parametrize("width", [1, 33, 128, 250, 512, 2730, 4096, 5000, 16300])
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_mxfp4_form_writes_the_stream_of_every_row(width, types):
    """The stream is one fp32 addition and one rounding, in every row, NaN among them too; the codes are those of that stream, formed apart from the call."""
    fo = _fo()
    dtype, stream_dtype = types
    for rows in (2, 9, 1100):
        x = (3.0 * torch.randn(rows, width, device=DEV)).to(dtype)
        residual = torch.randn(rows, width, device=DEV).to(stream_dtype)
        w = (1.0 + 0.3 * torch.randn(width, device=DEV)).to(dtype)
        x[rows // 2, width // 2] = float("nan")
        want = (x.float() + residual.float()).to(stream_dtype)
        q, s = fo.rms_norm_mxfp4(x, w, residual, eps=1e-5)
        torch.testing.assert_close(s, want, rtol=0, atol=0, equal_nan=True)
        codes = fo.mxfp4_quantize(fo.rms_norm(want.float(), w, eps=1e-5))
        assert torch.equal(q.scales, codes.scales) and torch.equal(q.codes, codes.codes), (width, types, rows)


def test_operands_without_memory_are_refused():
    """Wrappers and zeros that torch keeps no memory for have no address, which is how the C entry points are told that there is no weight: not ones in its place."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    fo = _fo()
    x, w = torch.randn(4, 40, device=DEV), torch.randn(40, device=DEV)
    with FakeTensorMode():
        fake, fake_x = torch.ones(40, device=DEV), torch.ones(4, 40, device=DEV)
    zeros, zeros_x = torch._efficientzerotensor(40, device=DEV), torch._efficientzerotensor((4, 40), device=DEV)
    for args in ((x, fake), (x, zeros), (fake_x, w), (zeros_x, w), (x, w, fake_x), (x, w, zeros_x)):
        for call in (fo.rms_norm, fo.rms_norm_mxfp4):
            with pytest.raises(NotImplementedError, match="in memory"):
                call(*args)
    with pytest.raises(NotImplementedError, match="in memory"):
        fo.linear_cross_entropy(x, fake_x, torch.zeros(4, dtype=torch.int64, device=DEV))
    with pytest.raises(NotImplementedError, match="in memory"):
        fo.embedding(torch.zeros(4, dtype=torch.int64, device=DEV), zeros_x)
