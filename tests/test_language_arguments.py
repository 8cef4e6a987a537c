"""What the embedding, the norm and the loss refuse before any device work, through their C entry points and through Python."""

import os
import threading

import pytest
import torch

import flashoptim_amd as fo
from flashoptim_amd import _autograd, _native

INVALID, UNSUPPORTED = -1, -2
SOME = 1 << 20    # an address that no call here gets to use
NAN = float("nan")


def test_norm_checks_its_arguments():
    lib = _native.lib()

    def call(x=SOME, x_dtype=1, rows=3, cols=5, residual=SOME, stream_dtype=1, weight=SOME, weight_dtype=0, eps=1e-6, out=SOME, y=SOME):
        return lib.fo_rms_norm(x, x_dtype, rows, cols, cols, residual, stream_dtype, cols, weight, weight_dtype, eps, out, y, None, None)

    def packed(scales=SOME, codes=SOME, **kw):
        a = {**dict(x=SOME, x_dtype=1, rows=3, cols=5, eps=1e-6), **kw}
        return lib.fo_rms_norm_mxfp4(a["x"], a["x_dtype"], a["rows"], a["cols"], a["cols"], None, 0, 0, None, 0, a["eps"], None, codes, scales, None)

    for bad in (dict(rows=-1), dict(cols=-1), dict(x_dtype=3), dict(x_dtype=-1), dict(stream_dtype=7), dict(weight_dtype=3), dict(eps=-1.0), dict(eps=NAN), dict(x=None), dict(y=None),
                dict(out=None)):
        assert call(**bad) == INVALID, bad
        assert lib.fo_last_error()
    assert call(stream_dtype=2) == UNSUPPORTED and call(cols=16385) == UNSUPPORTED and call(rows=1 << 31) == UNSUPPORTED
    assert call(rows=0, x=None, y=None) == 0 and call(cols=0, x=None, y=None) == 0
    for bad in (dict(scales=None), dict(codes=None), dict(codes=SOME + 8), dict(x=None), dict(x_dtype=4)):
        assert packed(**bad) == INVALID, bad


def test_norm_gradient_checks_its_arguments():
    lib = _native.lib()

    def call(s=SOME, stream_dtype=1, weight=SOME, weight_dtype=1, inverse=SOME, dy=SOME, x_dtype=1, rows=3, cols=5, dx=SOME, dresidual=None, dw=None):
        return lib.fo_rms_norm_backward(s, stream_dtype, cols, weight, weight_dtype, inverse, dy, x_dtype, cols, None, 0, rows, cols, dx, dresidual, dw, None, 0, None)

    for bad in (dict(s=None), dict(inverse=None), dict(dy=None), dict(dx=None), dict(rows=-1), dict(x_dtype=3), dict(weight=None, dw=SOME)):
        assert call(**bad) == INVALID, bad
    assert call(stream_dtype=2) == UNSUPPORTED and call(rows=0, s=None) == 0
    assert lib.fo_rms_norm_backward_workspace(-1, 5) == INVALID and lib.fo_rms_norm_backward_workspace(1, 16385) == UNSUPPORTED
    assert lib.fo_rms_norm_backward_workspace(0, 5) == 0


def test_embedding_checks_its_arguments():
    lib = _native.lib()

    def call(tokens=SOME, index=8, n=3, weight=SOME, dtype=1, vocabulary=7, cols=5, y=SOME):
        return lib.fo_embedding(tokens, index, n, weight, dtype, vocabulary, cols, cols, 1.0, y, None)

    def back(tokens=SOME, index=8, n=3, dy=SOME, dtype=1, vocabulary=7, cols=5, dw=SOME, workspace=SOME, size=1 << 30):
        return lib.fo_embedding_backward(tokens, index, n, dy, dtype, cols, vocabulary, cols, 1.0, -1, dw, workspace, size, None)

    for bad in (dict(index=2), dict(n=-1), dict(dtype=3), dict(vocabulary=-1), dict(cols=-1), dict(tokens=None)):
        assert call(**bad) == INVALID and back(**bad) == INVALID, bad
    assert call(weight=None) == INVALID and call(y=None) == INVALID
    for bad in (dict(dy=None), dict(dw=None), dict(workspace=None), dict(workspace=SOME + 128), dict(size=10)):
        assert back(**bad) == INVALID, bad
    for large in (dict(n=(1 << 25) + 1), dict(vocabulary=1 << 23), dict(cols=1 << 26), dict(vocabulary=(1 << 23) - 1, cols=1 << 15)):
        assert call(**large) == UNSUPPORTED and back(**large) == UNSUPPORTED, large
    assert call(n=0, tokens=None) == 0 and back(vocabulary=0, dw=None) == 0
    size = lib.fo_embedding_backward_workspace
    assert size(-1, 1, 1) == INVALID and size(0, 1000, 8) == 0
    # keys, a second array of them from the second run on, two rows a window of 16 from the second on
    assert size(16, 10, 8) == 256 and size(17, 10, 8) == 256 + 2 * 2 * 8 * 4 * 2 and size(512, 10, 8) == 4096 + 32 * 2 * 8 * 4
    assert size(513, 10, 8) == 2 * 4352 + -(-33 * 2 * 8 * 4 // 256) * 256


def test_loss_checks_its_arguments():
    lib = _native.lib()

    def call(x=SOME, dtype=1, tokens=3, weight=SOME, vocabulary=7, cols=5, targets=SOME, index=8, reduction=2, smoothing=0.0, loss=SOME, kept=SOME, workspace=SOME, size=1 << 40):
        return lib.fo_linear_cross_entropy(x, dtype, tokens, cols, weight, cols, vocabulary, cols, targets, index, -100, reduction, smoothing, loss, kept, workspace, size, None)

    def back(x=SOME, dtype=1, tokens=3, weight=SOME, vocabulary=7, cols=5, reduction=2, smoothing=0.0, kept=SOME, upstream=SOME, dx=SOME, workspace=SOME, size=1 << 40):
        return lib.fo_linear_cross_entropy_backward(x, dtype, tokens, cols, weight, cols, vocabulary, cols, reduction, smoothing, kept, upstream, 0, dx, None,
                                                    workspace, size, None)

    for bad in (dict(x=None), dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(weight=None), dict(vocabulary=-1), dict(cols=-1), dict(reduction=3),
                dict(reduction=-1), dict(smoothing=-0.5), dict(smoothing=1.5), dict(smoothing=NAN), dict(kept=None), dict(workspace=None), dict(workspace=SOME + 64), dict(size=100)):
        assert call(**bad) == INVALID and back(**bad) == INVALID, bad
    assert call(loss=None) == INVALID and call(targets=None) == INVALID and call(index=1) == INVALID and back(upstream=None) == INVALID and back(dx=None) == INVALID
    for other in (dict(tokens=0), dict(cols=0), dict(vocabulary=0), dict(tokens=(1 << 20) + 1), dict(cols=65537), dict(vocabulary=(1 << 24) + 1)):
        assert call(**other) == UNSUPPORTED and back(**other) == UNSUPPORTED, other

    def forward(dtype, tokens, cols, vocabulary, smoothing=0.0, x=SOME, x_stride=None, weight=SOME, weight_stride=None):
        return lib.fo_linear_cross_entropy_workspace(x, dtype, tokens, x_stride or cols, weight, weight_stride or cols, vocabulary, cols, smoothing)

    def backward(dtype, tokens, cols, vocabulary, dx=1, dw=1, weight=SOME):
        return lib.fo_linear_cross_entropy_backward_workspace(SOME, dtype, tokens, cols, weight, cols, vocabulary, cols, dx, dw)

    assert forward(1, -1, 5, 7) == INVALID and forward(1, 0, 5, 7) == UNSUPPORTED and backward(5, 3, 5, 7) == INVALID
    # some bytes a row of a tile's part forward, a piece's gradient of 2^27 values, x and sums between pieces backward: not the logits, and not the weight
    logits = 8192 * 128256 * 2
    assert forward(1, 8192, 4096, 128256) < logits // 20 and backward(1, 8192, 4096, 128256) < logits // 4
    assert backward(1, 8192, 4096, 128256, 1, 0) > backward(1, 8192, 4096, 128256, 0, 1)    # the sums
    assert forward(1, 8192, 4096, 128256, smoothing=0.1) > forward(1, 8192, 4096, 128256)
    # what cannot be read in place is laid out
    weight = 128256 * 4096 * 2
    for other in (dict(weight=SOME + 2), dict(weight_stride=4097)):
        assert forward(1, 8192, 4096, 128256, **other) >= forward(1, 8192, 4096, 128256) + weight, other
    assert forward(1, 8192, 4096, 128256, x=SOME + 2) >= forward(1, 8192, 4096, 128256) + 8192 * 4096 * 2


def test_without_a_gpu():
    x = torch.zeros(3, 8)
    for call in (lambda: fo.rms_norm(x), lambda: fo.rms_norm_mxfp4(x), lambda: fo.embedding(torch.zeros(2, dtype=torch.int64), x),
                 lambda: fo.linear_cross_entropy(x, x, torch.zeros(3, dtype=torch.int64)), lambda: fo.FlashRMSNorm(8)(x),
                 lambda: fo.FlashEmbedding(4, 8)(torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(NotImplementedError):
            call()


def test_modules_check_what_they_are_made_of():
    table = torch.randn(7, 5, dtype=torch.bfloat16)
    frozen, free = fo.FlashEmbedding.from_pretrained(table, scale=2.0), fo.FlashEmbedding.from_pretrained(table, freeze=False, padding_idx=-1)
    assert torch.equal(frozen.weight, table) and not frozen.weight.requires_grad and frozen.scale == 2.0 and frozen.padding_idx is None
    assert free.weight.requires_grad and free.padding_idx == 6 and (free.num_embeddings, free.embedding_dim) == (7, 5)
    assert frozen.weight.data_ptr() == table.data_ptr()
    with pytest.raises(ValueError):
        fo.FlashEmbedding.from_pretrained(table[0])
    with pytest.raises(TypeError):
        fo.FlashRMSNorm((4, 5))
    norm = fo.FlashRMSNorm(8, elementwise_affine=False)
    with pytest.raises(ValueError):
        norm(torch.randn(3, 4))
    with pytest.raises(ValueError):
        norm(torch.tensor(1.0))


@pytest.mark.skipif(not os.path.exists(_autograd.library_path()), reason="the C++ calls are not built")
def test_calls_built_for_another_interface_are_left_out(monkeypatch):
    names = ("rms_norm", "rms_norm_mxfp4", "embedding", "linear_cross_entropy")
    for name in (*names, "_module"):
        monkeypatch.setattr(_autograd, name, None)
    monkeypatch.delenv("FLASHOPTIM_NO_HOSTSCAN", raising=False)
    result, arguments = _native.SIGNATURES["fo_embedding"]
    with monkeypatch.context() as other:
        other.setitem(_native.SIGNATURES, "fo_embedding", (result, arguments[:-1]))
        _autograd._load()
        assert all(getattr(_autograd, name) is None for name in names) and _autograd._module is None
    _autograd._load()
    assert all(getattr(_autograd, name) is not None for name in names)


def test_first_calls_of_several_threads(monkeypatch):
    """Threads that call first, together: every one finds the module bound, or binds it."""
    bound, failed, together, lib = [], [], threading.Barrier(4, timeout=30), _native.lib()

    class Module:
        def bind(self, addresses):
            bound.append(addresses)

    def load():
        together.wait()    # every thread has seen that nothing is bound
        return lib

    monkeypatch.setattr(_autograd, "_module", Module())
    monkeypatch.setattr(_native, "lib", load)

    def call():
        try:
            _autograd.bind()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=call) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and _autograd._module is None
    assert bound and all(b == bound[0] and all(b.values()) for b in bound)


def test_the_loss_gradient_takes_a_bounded_workspace():
    """2^28 bytes of G, up to 256 words more of every token, since pieces are whole multiples of that; beside it dx in fp32 between pieces, or in parts where rows are few, two
    numbers a token, and fp32 operands that are laid out."""
    lib = _native.lib()
    for dtype, bytes_a_word in ((0, 6), (1, 2), (2, 2)):    # of fp32 at most three parts
        for tokens in (1, 1000, 8192, 50000, 300000, 1 << 20):
            for vocabulary in (33, 128256, 1 << 24):
                size = lib.fo_linear_cross_entropy_backward_workspace(SOME, dtype, tokens, 64, SOME, 64, vocabulary, 64, 1, 0)
                operands = 0 if dtype else 6 * 64 * (tokens + 64 + (1 << 28) // (6 * tokens) + 512)    # fp32 in parts: x and a piece of the matrix
                sums, parts = 4 * 64 * tokens, 4 * 64 * tokens * 32 if tokens <= 8192 else 0
                assert 0 < size <= (1 << 28) + 257 * tokens * bytes_a_word + sums + parts + 8 * tokens + operands + (1 << 20), (dtype, tokens, vocabulary)
