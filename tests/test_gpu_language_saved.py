"""GPU tests of the embedding's, the norm's and the loss's backward passes when what was saved for them has been through a user's hands: hooks on saved tensors."""

import threading

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(params=["nodes", "python"], autouse=True)
def host(request, monkeypatch):
    """Every test through the C++ calls and nodes, and through the Python ones that stand in for them."""
    from flashoptim_amd import _autograd

    _autograd.bind()
    assert _autograd.rms_norm and _autograd.embedding and _autograd.linear_cross_entropy
    if request.param == "python":
        for name in ("rms_norm", "rms_norm_mxfp4", "embedding", "linear_cross_entropy"):
            monkeypatch.setattr(_autograd, name, None)
    return request.param


def _fo():
    import flashoptim_amd

    return flashoptim_amd


def _through_bf16():
    """Hooks that hold floating-point tensors in bf16."""
    return saved_tensors_hooks(lambda t: (t.dtype, t.to(BF16) if t.is_floating_point() else t), lambda packed: packed[1].to(packed[0]))


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_labels_are_not_converted(tokens):
    """x and the matrix are bf16 already, so hooks that hold floating-point tensors in bf16 change nothing: the labels, of which bf16 holds few, are not floating-point."""
    fo = _fo()
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x, w = torch.randn(tokens, 64, generator=g, device=DEV).to(BF16).requires_grad_(), torch.randn(70001, 64, generator=g, device=DEV).to(BF16).requires_grad_()
    target = torch.randint(69000, 70001, (tokens,), generator=g, device=DEV)
    target[2::5] = -100
    want = torch.autograd.grad(fo.linear_cross_entropy(x, w, target), (x, w))
    with _through_bf16():
        loss = fo.linear_cross_entropy(x, w, target)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), want))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_labels_beyond_the_vocabulary_are_no_addresses(dtype):
    """The C entry point with labels that are none of its own: their rows have no target, the others are as they were."""
    from flashoptim_amd import _native

    lib, code, (n, k, v) = _native.lib(), _native.DTYPE_CODE[dtype], (9, 64, 130)
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w = torch.randn(n, k, generator=g, device=DEV).to(dtype), torch.randn(v, k, generator=g, device=DEV).to(dtype)
    target, up, loss = torch.randint(0, v, (n,), generator=g, device=DEV), torch.ones((), device=DEV), torch.empty((), device=DEV)
    kept = torch.empty(_native.LOSS_NUMBERS_A_TOKEN * n + 1, dtype=torch.int32, device=DEV)
    stream = _native.current_stream_ptr(x.device)
    space = torch.empty(lib.fo_linear_cross_entropy_workspace(x.data_ptr(), code, n, k, w.data_ptr(), k, v, k, 0.0), dtype=torch.uint8, device=DEV)
    assert lib.fo_linear_cross_entropy(x.data_ptr(), code, n, k, w.data_ptr(), k, v, k, target.data_ptr(), 8, -100, 1, 0.0, loss.data_ptr(), kept.data_ptr(), space.data_ptr(),
                                       space.numel(), stream) == 0
    space = torch.empty(lib.fo_linear_cross_entropy_backward_workspace(x.data_ptr(), code, n, k, w.data_ptr(), k, v, k, 1, 0), dtype=torch.uint8, device=DEV)

    def dx():
        out = torch.empty_like(x)
        assert lib.fo_linear_cross_entropy_backward(x.data_ptr(), code, n, k, w.data_ptr(), k, v, k, 1, 0.0, kept.data_ptr(), up.data_ptr(), 0, out.data_ptr(), None, space.data_ptr(),
                                                    space.numel(), stream) == 0
        return out

    clean, others = dx(), torch.tensor([0, 1, 3, 5, 7, 8], device=DEV)
    labels = kept[2 * n + 1:]
    assert torch.equal(labels, target.int())
    labels[2], labels[4], labels[6] = v, 2 ** 31 - 1, 131072
    got = dx()
    assert torch.equal(got[others], clean[others])
    p = torch.softmax(x.double() @ w.double().t(), 1)    # 64 products of fp32, probabilities rounded to the type, the result too: 2^-6 of the magnitudes' sum is far above
    assert bool(((got.double() - p @ w.double()).abs() <= 2.0 ** -6 * (p @ w.double().abs()))[[2, 4, 6]].all())


def _laid_out(how):
    """Hooks that give back the same values, another way round in memory."""

    def other(t):
        if t.dim() == 0 or t.numel() == 0:
            return t.clone()
        if how == "turned":    # the last axis is the one that lies apart
            return t.transpose(0, -1).contiguous().transpose(0, -1)
        if how == "apart":     # neither values nor rows are neighbours
            wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1] + 3, dtype=t.dtype, device=t.device)
            wide[..., 1:2 * t.shape[-1]:2] = t
            return wide[..., 1:2 * t.shape[-1]:2]
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, dtype=t.dtype, device=t.device)
        wide[..., 2:-3] = t
        return wide[..., 2:-3]

    return saved_tensors_hooks(lambda t: t.clone(), other)


def _calls():
    """Each operator with its leaves, matrices and batches of them."""
    fo = _fo()
    g = torch.Generator(device=DEV).manual_seed(5)

    def values(*shape, dtype=BF16):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype).requires_grad_()

    target = torch.randint(0, 33, (4, 6), generator=g, device=DEV)
    table, x, r, scale, dy = values(33, 40), values(4, 6, 40), values(4, 6, 40, dtype=F32), values(40), values(4, 6, 40).detach()
    flat, flat_r = values(24, 40), values(24, 40, dtype=F32)
    yield "embedding", lambda: fo.embedding(target, table), (table,), dy
    yield "embedding of a row", lambda: fo.embedding(target[0], table), (table,), dy[0]
    yield "norm", lambda: fo.rms_norm(x, scale), (x, scale), dy
    yield "norm with a residual", lambda: fo.rms_norm(x, scale, r)[0], (x, scale, r), dy
    yield "norm of a matrix", lambda: fo.rms_norm(flat, scale), (flat, scale), dy.view(24, 40)
    yield "norm of a matrix with a residual", lambda: fo.rms_norm(flat, scale, flat_r)[0], (flat, scale, flat_r), dy.view(24, 40)
    yield "loss", lambda: fo.linear_cross_entropy(x, table, target, label_smoothing=0.1), (x, table), None
    yield "loss of a matrix", lambda: fo.linear_cross_entropy(flat, table, target.view(24)), (flat, table), None


@pytest.mark.parametrize("how", ["turned", "apart", "rows apart"])
def test_what_hooks_lay_out_anew_is_read_right(how):
    for what, call, leaves, dy in _calls():
        want = torch.autograd.grad(call(), leaves, dy)
        with _laid_out(how):
            out = call()
        got = torch.autograd.grad(out, leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (how, what)


def test_other_tensors_than_those_that_were_saved_are_refused():
    for change in (lambda t: t.double() if t.is_floating_point() else t.short(), lambda t: t[:-1], lambda t: t.unsqueeze(0), lambda t: t.cpu()):
        for what, call, leaves, dy in _calls():
            with saved_tensors_hooks(lambda t: t, change):
                out = call()
            with pytest.raises(RuntimeError, match="hook on saved tensors"):
                torch.autograd.grad(out, leaves, dy)


def test_backward_passes_of_one_graph_in_several_threads():
    """Of a graph that is kept every thread gets the gradients; of one that is not, each gets them or hears that they are gone."""
    for what, call, leaves, dy in _calls():
        out = call()
        want = torch.autograd.grad(out, leaves, dy, retain_graph=True)
        torch.cuda.synchronize()
        for keep in (True, False):
            got, gone, other = [], [], []

            def backward():
                for _ in range(10):
                    try:
                        got.append(torch.autograd.grad(out, leaves, dy, retain_graph=keep))
                    except RuntimeError as e:
                        (gone if "second time" in str(e) or "freed" in str(e) else other).append(e)

            threads = [threading.Thread(target=backward) for _ in range(4)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            assert not other and len(got) + len(gone) == 40 and len(got) >= (40 if keep else 1), (what, other)
            assert all(torch.equal(a, b) for g in got for a, b in zip(g, want)), what
