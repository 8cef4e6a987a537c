"""The embedding, the norm and the loss together, as a model uses them: gradients of the whole against 64 bits, training and serving, streams, threads, graphs,
tied weights, the optimizers' masters.

What the whole is allowed: each step's own tests hold it to its formula; here what counts is that they fit together, so a gradient of the whole is compared with
the same model in 64 bits by its norm.  In fp32 that is 1e-5 (a few thousand roundings of 2^-24 that add up at random, and some that do not); in bf16 each of the 8 tensors on
the way is rounded to 2^-8 of itself at most, 2^-9 at random, so 8^(1/2) 2^-9 at random and 8 2^-9 at most.
"""

import threading

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
VOCABULARY, WIDTH = 301, 96


def _fo():
    import flashoptim_amd

    return flashoptim_amd


class Model(nn.Module):
    """Two residual layers between an embedding and an output matrix that is the same one."""

    def __init__(self, dtype):
        fo = _fo()
        super().__init__()
        self.embed = fo.FlashEmbedding(VOCABULARY, WIDTH, padding_idx=0, scale=3.0, device=DEV, dtype=dtype)
        self.norms = nn.ModuleList(fo.FlashRMSNorm(WIDTH, eps=1e-5, device=DEV, dtype=dtype) for _ in range(3))
        self.layers = nn.ModuleList(nn.Linear(WIDTH, WIDTH, bias=False, device=DEV, dtype=dtype) for _ in range(2))

    def forward(self, tokens, target):
        fo = _fo()
        branch = self.embed(tokens)
        y, stream = self.norms[0](branch), branch
        for norm, layer in zip(self.norms[1:], self.layers):
            y, stream = norm(F.silu(layer(y)), stream)
        return fo.linear_cross_entropy(y, self.embed.weight, target, label_smoothing=0.1)


def _reference(model, tokens, target):
    """The same in 64 bits, with the parameters' gradients."""
    p = {n: t.detach().double().requires_grad_() for n, t in model.named_parameters()}
    norm = lambda x, w: x * (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w  # noqa: E731
    table = p["embed.weight"]
    branch = 3.0 * torch.where((tokens == 0).unsqueeze(-1), table[0].detach(), table[tokens])
    y, stream = norm(branch, p["norms.0.weight"]), branch
    for i in range(2):
        stream = stream + F.silu(y @ p[f"layers.{i}.weight"].t())
        y = norm(stream, p[f"norms.{i + 1}.weight"])
    loss = F.cross_entropy((y @ table.t()).flatten(0, 1), target.flatten().long(), label_smoothing=0.1)
    return loss, dict(zip(p, torch.autograd.grad(loss, p.values())))


def _data(seed, batch=7, length=33):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(1, VOCABULARY, (batch, length), generator=g)
    target = torch.randint(0, VOCABULARY, (batch, length), generator=g)
    for i in range(batch):    # padded rows of the batch
        tokens[i, length - i:], target[i, length - i:] = 0, -100
    return tokens.to(DEV), target.to(DEV)


@pytest.mark.parametrize("dtype,allowed", [(torch.float32, 1e-5), (torch.bfloat16, 8 * 2.0 ** -9), (torch.float16, 8 * 2.0 ** -12)])
def test_gradients_of_the_whole(dtype, allowed):
    torch.manual_seed(0)
    model = Model(dtype)
    tokens, target = _data(1)
    loss = model(tokens, target)
    loss.backward()
    want, grads = _reference(model, tokens, target)
    assert abs(float(loss) - float(want)) < allowed * float(want)
    for name, p in model.named_parameters():
        far = float((p.grad.double() - grads[name]).norm() / grads[name].norm())
        assert far < allowed, (name, far)


def test_training_with_the_optimizers():
    """Masters in 24 bits, steps as gradients arrive: a run goes through, and twice the same."""
    fo = _fo()
    ends = []
    for _ in range(2):
        torch.manual_seed(0)
        model = Model(torch.bfloat16)
        opt = fo.FlashAdamW(model.parameters(), lr=1e-2, weight_decay=0.0, master_weight_bits=24)
        for step in range(4):
            model(*_data(step)).backward()
            opt.step()
            opt.zero_grad()
        ends.append([p.detach().clone() for p in model.parameters()])
        assert all(bool(p.isfinite().all()) for p in ends[-1])
    assert all(torch.equal(a, b) for a, b in zip(*ends))


def test_a_token_at_a_time_equals_all_at_once():
    """Rows do not know of one another: what a batch gets is what its rows get alone, to the bit."""
    fo = _fo()
    torch.manual_seed(0)
    for dtype in (torch.float32, torch.bfloat16):
        weight, table = torch.randn(WIDTH, device=DEV).to(dtype), torch.randn(VOCABULARY, WIDTH, device=DEV).to(dtype)
        tokens, target = _data(2)
        rows = fo.embedding(tokens, table, scale=2.0).view(-1, WIDTH)
        stream = torch.randn(rows.shape, device=DEV).to(dtype)
        y, s = fo.rms_norm(rows, weight, stream)
        q, _ = fo.rms_norm_mxfp4(rows, weight, stream)
        for i in (0, 5, 100, 230):
            one = fo.embedding(tokens.view(-1)[i], table, scale=2.0)
            assert torch.equal(one, rows[i])
            y1, s1 = fo.rms_norm(one.view(1, -1), weight, stream[i:i + 1])
            q1, _ = fo.rms_norm_mxfp4(one.view(1, -1), weight, stream[i:i + 1])
            assert torch.equal(y1[0], y[i]) and torch.equal(s1[0], s[i]) and torch.equal(q1.codes[0], q.codes[i]) and torch.equal(q1.scales[0], q.scales[i])


def test_on_another_stream_and_in_threads():
    """Calls on streams of their own, from two threads at once, give what one call alone gives."""
    torch.manual_seed(0)
    model = Model(torch.bfloat16)
    data = [_data(i) for i in range(2)]
    params = list(model.parameters())
    want = [[t.clone() for t in torch.autograd.grad(model(*d), params)] for d in data]
    got, errors = [None, None], []
    torch.cuda.synchronize()

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[i] = torch.autograd.grad(model(*data[i]), params)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_captured_step():
    """A whole step's forward and backward pass in a graph, replayed between eager ones on new data."""
    torch.manual_seed(0)
    model = Model(torch.bfloat16)
    params = list(model.parameters())
    tokens, target = _data(0)

    def step():
        loss = model(tokens, target)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(1, 4):
        more_tokens, more_target = _data(seed)
        tokens.copy_(more_tokens)
        target.copy_(more_target)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), seed


def test_two_graphs_share_nothing():
    fo = _fo()
    torch.manual_seed(0)
    x, w = torch.randn(200, 64, device=DEV, requires_grad=True), torch.randn(500, 64, device=DEV, requires_grad=True)
    targets = [torch.randint(0, 500, (200,), device=DEV) for _ in range(2)]
    run = lambda t: torch.autograd.grad(fo.linear_cross_entropy(x, w, t), (x, w))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(targets[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for t in targets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(t))
    want = [run(t) for t in targets]
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_rows_behind_the_results_are_left_alone():
    """Results that are parts of larger buffers, through the C entry points: nothing is written around them."""
    from flashoptim_amd import _native

    fo = _fo()
    lib, s = _native.lib(), _native.current_stream_ptr(torch.device(DEV))
    x, w = torch.randn(5, 24, device=DEV), torch.randn(11, 24, device=DEV)
    target = torch.tensor([1, 2, 3, 10, 0], device=DEV)
    buffers = {n: torch.full((size + 512,), 77.0, device=DEV) for n, size in dict(y=120, loss=5, kept=16, dx=120, dw=264, rows=120, table=264).items()}
    at = {n: b.data_ptr() + 1024 for n, b in buffers.items()}
    assert lib.fo_rms_norm(x.data_ptr(), 0, 5, 24, 24, None, 0, 0, None, 0, 1e-6, None, at["y"], None, s) == 0
    size = lib.fo_linear_cross_entropy_workspace(x.data_ptr(), 0, 5, 24, w.data_ptr(), 24, 11, 24, 0.0)
    space = torch.empty(size, dtype=torch.uint8, device=DEV)
    assert lib.fo_linear_cross_entropy(x.data_ptr(), 0, 5, 24, w.data_ptr(), 24, 11, 24, target.data_ptr(), 8, -100, 0, 0.0, at["loss"], at["kept"], space.data_ptr(), size, s) == 0
    size = lib.fo_linear_cross_entropy_backward_workspace(x.data_ptr(), 0, 5, 24, w.data_ptr(), 24, 11, 24, 1, 1)
    back, ones = torch.empty(size, dtype=torch.uint8, device=DEV), torch.ones(5, device=DEV)
    assert lib.fo_linear_cross_entropy_backward(x.data_ptr(), 0, 5, 24, w.data_ptr(), 24, 11, 24, 0, 0.0, at["kept"], ones.data_ptr(), 1, at["dx"], at["dw"], back.data_ptr(), size, s) == 0
    assert lib.fo_embedding(target.data_ptr(), 8, 5, w.data_ptr(), 0, 11, 24, 24, 1.0, at["rows"], s) == 0
    size = lib.fo_embedding_backward_workspace(5, 11, 24)
    keys = torch.empty(size, dtype=torch.uint8, device=DEV)
    assert lib.fo_embedding_backward(target.data_ptr(), 8, 5, x.data_ptr(), 0, 24, 11, 24, 1.0, -1, at["table"], keys.data_ptr(), size, s) == 0
    torch.cuda.synchronize()
    for n, b in buffers.items():
        assert bool((b[:256] == 77.0).all()) and bool((b[-256:] == 77.0).all()), n
    leaves = [x.requires_grad_(), w.requires_grad_()]
    loss = fo.linear_cross_entropy(*leaves, target, reduction="none")
    dx, dw = torch.autograd.grad(loss, leaves, ones)
    assert torch.equal(buffers["loss"][256:261], loss) and torch.equal(buffers["dx"][256:-256], dx.flatten()) and torch.equal(buffers["dw"][256:-256], dw.flatten())
    assert torch.equal(buffers["rows"][256:-256], w[target].flatten()) and torch.equal(buffers["y"][256:-256], fo.rms_norm(x).flatten())


def test_cast_models_keep_their_head_in_fp32():
    """cast_model with the output matrix kept in fp32: hidden states go to it in fp32, and its gradient is fp32's."""
    fo = _fo()
    torch.manual_seed(0)
    head = nn.Linear(WIDTH, VOCABULARY, bias=False, device=DEV)
    body = nn.Linear(WIDTH, WIDTH, device=DEV)
    model = nn.ModuleDict(dict(body=body, head=head))
    fo.cast_model(model, full_precision_layers=["head"])
    x = torch.randn(50, WIDTH, device=DEV).to(torch.bfloat16)
    target = torch.randint(0, VOCABULARY, (50,), device=DEV)
    y = body(x)
    loss = fo.linear_cross_entropy(y.float(), head.weight, target)
    loss.backward()
    assert head.weight.grad.dtype == torch.float32 and body.weight.grad.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="type"):
        fo.linear_cross_entropy(y, head.weight, target)


@pytest.fixture(params=["nodes", "python"])
def host(request, monkeypatch):
    """Through the C++ calls and nodes, and through the Python ones that stand in for them."""
    from flashoptim_amd import _autograd

    _autograd.bind()
    if request.param == "python":
        for name in ("rms_norm", "rms_norm_mxfp4", "embedding", "linear_cross_entropy"):
            monkeypatch.setattr(_autograd, name, None)
    return request.param


def test_under_checkpoints_and_hooks_on_what_is_saved(host):
    from torch.utils.checkpoint import checkpoint

    model = Model(torch.bfloat16)
    tokens, target = _data(11)
    parameters = list(model.parameters())
    want = torch.autograd.grad(model(tokens, target), parameters)

    def same(got):
        return all(torch.equal(a, b) for a, b in zip(want, got))

    assert same(torch.autograd.grad(checkpoint(model, tokens, target, use_reentrant=False), parameters))
    with torch.autograd.graph.save_on_cpu():
        loss = model(tokens, target)
    assert same(torch.autograd.grad(loss, parameters))
    checkpoint(lambda table: model(tokens, target) + 0.0 * table.sum(), model.embed.weight, use_reentrant=True).backward()
    assert same([p.grad for p in parameters])
    # a graph that is kept gives the same again, and adds up
    loss = model(tokens, target)
    for _ in range(2):
        loss.backward(retain_graph=True)
    for p, g in zip(parameters, want):    # two additions, each rounded by at most half a step of at most three times the gradient
        assert (p.grad.float() - 3 * g.float()).abs().max() <= 3 * 2.0 ** -7 * g.float().abs().max()


def test_modes_without_a_graph_and_transforms(host):
    fo = _fo()
    model = Model(torch.bfloat16)
    tokens, target = _data(12)
    loss = model(tokens, target)
    with torch.no_grad():
        assert torch.equal(model(tokens, target), loss)
    with torch.inference_mode():
        assert torch.equal(model(tokens, target), loss)
        y, stream = fo.rms_norm(torch.ones(3, 8, device=DEV), None, torch.ones(3, 8, device=DEV))
        assert y.is_inference() and stream.is_inference()
    x, w = torch.randn(5, 8, device=DEV), torch.randn(9, 8, device=DEV)
    at = torch.tensor([1, 2, 3, 4, 5], device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):    # nothing is converted
        assert fo.rms_norm(x).dtype == torch.float32 and fo.linear_cross_entropy(x, w, at).dtype == torch.float32
    for f in (lambda t: fo.rms_norm(t).sum(), lambda t: fo.linear_cross_entropy(t, w, at), lambda t: fo.embedding(at, t).sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(f)(x)
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x.expand(2, 5, 8).contiguous())
