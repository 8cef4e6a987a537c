"""The operators of low-precision training that this package adds to its optimizer step, as timed cases.

Two families that meet in one training step: the hidden matrices of a network are multiplied in microscaled 4-bit floating
point (MXFP4: groups of 32 E2M1 values that share an E8M0 scale), forward and backward, and their gradients are
orthogonalised by Newton-Schulz products before they change the weights, as the Muon optimizer does.

A case is one call.  ``task`` says which:

* ``ns``     a stack of matrices through the Newton-Schulz iteration;
* ``muon``   one optimizer step over a list of matrices: 8-bit momentum, orthogonalised update, masters of more bits than
             the weights;
* ``quant``  a matrix into MXFP4, along its rows, its columns or both, and back;
* ``train``  a linear layer in MXFP4: output, gradient of the input, gradient of the weight;
* ``serve``  a few tokens through a weight that is held in MXFP4.

Gradients have a few strong directions above noise, activations some channels far larger than the rest, weights are normal.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_WIDTH = {"bf16": 2, "fp16": 2, "fp32": 4}
_GROUP = 32                                   # values that share one scale, here and in the 8-bit momentum
_ALIGN = 512                                  # elements between the starts of carved tensors
_STEPS = 5
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_NORM_EPS = 1e-7
_LR, _MOMENTUM, _DECAY = 2e-4, 0.95, 0.1      # a run in its middle, its learning rate on the way down


# ------------------------------------------------------------------------------------------------- the cases


def _ns(name, dtype, batch, rows, cols, view="whole"):
    return dict(name=name, task="ns", dtype=dtype, batch=batch, rows=rows, cols=cols, view=view)


def _muon(name, dtype, master, layers, hidden, ffn, kv, quantize=True):
    return dict(name=name, task="muon", dtype=dtype, master=master, quantize=quantize, layers=layers, hidden=hidden, ffn=ffn, kv=kv)


def _quant(name, dtype, rows, cols, along):
    return dict(name=name, task="quant", dtype=dtype, rows=rows, cols=cols, along=along)


def _train(name, dtype, tokens, inner, outer):
    return dict(name=name, task="train", dtype=dtype, tokens=tokens, inner=inner, outer=outer)


def _serve(name, dtype, tokens, inner, outer):
    return dict(name=name, task="serve", dtype=dtype, tokens=tokens, inner=inner, outer=outer)


def listed():
    return [
        # the first layer of the smallest program (a two-layer perceptron): one matrix, latency alone
        _ns("ns-mlp", "bf16", 1, 256, 128),
        # key projections of a small model with widths that are no powers of two, fp32 gradients cut out of fused ones
        _ns("ns-kv-odd", "fp32", 8, 250, 1000, "columns"),
        # the largest matrix of the 8B-parameter transformer's layer that the package's benchmark steps
        _ns("ns-ffn", "bf16", 1, 14336, 4096),
        # one whole layer of that transformer, default masters
        _muon("muon-block", "bf16", 24, 1, 4096, 14336, 1024),
        # four layers of a small model in fp16 with 32-bit masters, odd widths
        _muon("muon-odd", "fp16", 32, 4, 1000, 2730, 250),
        # a weight of that layer for the next step: what the product contracts over in the forward and in the backward pass
        _quant("quant-weight", "bf16", 14336, 4096, "both"),
        # activations of a small model, a ragged number of tokens
        _quant("quant-odd", "fp16", 1003, 2730, "rows"),
        # the layer's widest product over a batch of 4096 tokens, forward and backward
        _train("train-ffn", "bf16", 4096, 4096, 14336),
        # the same of the small model, nothing a multiple of a tile
        _train("train-odd", "fp16", 1003, 1000, 2730),
        # one token through the down projection
        _serve("serve-one", "bf16", 1, 14336, 4096),
        # a batch of sequences, one token each, through the up projection
        _serve("serve-batch", "bf16", 16, 4096, 14336),
        # a few drafted tokens in a small model
        _serve("serve-odd", "fp16", 5, 1000, 2730),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(2 ** rng.uniform(math.log2(lo), math.log2(hi))))

    task = rng.choice(["ns", "ns", "muon", "muon", "quant", "train", "train", "serve", "serve"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if task == "ns":
        while True:
            batch, rows, cols = log(1, 64), log(16, 14336), log(16, 14336)
            if batch * rows * cols <= 14336 * 4096 and min(rows, cols) <= 4096:
                break
        case = _ns("", dtype, batch, rows, cols, rng.choice(["whole", "whole", "columns", "transposed"]))
    elif task == "muon":
        hidden = log(96, 4096)
        master = 0 if dtype == "fp32" else rng.choice([24, 24, 32])
        case = _muon("", dtype, master, rng.randint(1, 4) if hidden < 2048 else 1, hidden, min(14336, int(hidden * rng.uniform(2, 3.5))),
                     max(16, hidden // rng.choice([1, 4, 8])), rng.random() < 0.85)
    elif task == "quant":
        while True:
            rows, cols = log(1, 14336), log(16, 14336)
            if rows * cols <= 14336 * 4096:
                break
        case = _quant("", dtype, rows, cols, rng.choice(["rows", "columns", "both"]))
    elif task == "train":
        case = _train("", rng.choice(["bf16", "fp16"]), log(1, 4096), log(32, 4096), log(32, 14336))
    else:
        case = _serve("", rng.choice(["bf16", "fp16"]), log(1, 64), log(32, 14336), log(32, 4096))
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------- inputs


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _gradients(g, batch, rows, cols, size):
    """Matrices with a few strong directions above noise, `size` about the magnitude of an entry."""
    strong = max(1, min(rows, cols) // 16)
    left, right = _normal(g, batch, rows, strong), _normal(g, batch, strong, cols)
    decay = torch.arange(1, strong + 1, device="cuda", dtype=torch.float32).rsqrt()
    return size * (torch.bmm(left * decay, right) / math.sqrt(strong) + 0.25 * _normal(g, batch, rows, cols))


def _activations(g, tokens, width):
    return _normal(g, tokens, width) * (1.0 + 7.0 * (torch.rand(width, generator=g, device="cuda") < 0.01))


def _muon_shapes(case):
    h, f, kv = case["hidden"], case["ffn"], case["kv"]
    return [(h, h), (kv, h), (kv, h), (h, h), (f, h), (f, h), (h, f)] * case["layers"]


def _starts(shapes):
    """Where each of the tensors that are carved from one flat buffer begins, and the buffer's length."""
    starts, total = [], 0
    for r, c in shapes:
        starts.append(total)
        total += -(-r * c // _ALIGN) * _ALIGN
    return starts, total


def _ecc_bytes(case):
    return max(0, case["master"] // 8 - _WIDTH[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, task = _DTYPES[case["dtype"]], case["task"]
    state = dict(case=case)
    if task == "ns":
        batch, rows, cols = case["batch"], case["rows"], case["cols"]
        if case["view"] == "transposed":
            state["x"] = _gradients(g, batch, cols, rows, 1e-3).to(dtype).transpose(1, 2)
        else:
            more = 24 if case["view"] == "columns" else 0    # the matrices are columns of wider ones
            state["x"] = _gradients(g, batch, rows, cols + more, 1e-3).to(dtype)[:, :, more // 2:more // 2 + cols]
    elif task == "quant":
        state["x"] = _activations(g, case["rows"], case["cols"]).to(dtype)
    elif task == "train":
        state["x"] = _activations(g, case["tokens"], case["inner"]).to(dtype)
        state["weight"] = (0.02 * _normal(g, case["outer"], case["inner"])).to(dtype)
        state["dy"] = _gradients(g, 1, case["tokens"], case["outer"], 1e-2)[0].to(dtype)
    elif task == "serve":
        state["x"] = _activations(g, case["tokens"], case["inner"]).to(dtype)
        values, scales = _mx_parts(0.02 * _normal(g, case["outer"], case["inner"]))
        # the stored form: two codes in a byte, the first in the low half, rows of whole 128-value blocks
        half = (values.abs() * 2.0).to(torch.int64)
        codes = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], device="cuda")[half] + 8 * (values < 0).long()
        state["codes"] = (codes[:, 0::2] + 16 * codes[:, 1::2]).to(torch.uint8)
        state["scales"] = (scales + 127).to(torch.uint8)
    else:
        _prepare_muon(state, case, g, dtype)
    return state


def _prepare_muon(state, case, g, dtype):
    shapes = _muon_shapes(case)
    starts, total = _starts(shapes)
    param = (0.02 * _normal(g, total)).to(dtype)
    grad, momentum = torch.zeros(total, device="cuda", dtype=dtype), torch.zeros(total, device="cuda")
    for at, (r, c) in zip(starts, shapes):
        size = 1e-3 / math.sqrt(r)
        both = _gradients(g, 2, r, c, size)
        grad[at:at + r * c] = both[0].reshape(-1)
        momentum[at:at + r * c] = (0.4 * both[0] + 0.1 * both[1]).reshape(-1)
    state.update(shapes=shapes, starts=starts, param=param, grad=grad)
    if case["quantize"]:
        state["codes"], state["scales"] = _moment_codes(momentum)
    else:
        state["momentum"] = momentum.to(dtype)
    ecc = _ecc_bytes(case)
    if ecc:
        top, kind = (127, torch.int8) if ecc == 1 else (32767, torch.int16)
        state["ecc"] = torch.randint(-top, top + 1, (total,), generator=g, device="cuda", dtype=kind)
    if not own:
        return
    # the optimizer that a training program keeps, in the middle of its run
    import warnings

    import flashoptim_amd as fo
    from flashoptim_amd.state import _MaybeQuantizedTensor

    carved = [slice(at, at + r * c) for at, (r, c) in zip(starts, shapes)]
    params = [torch.nn.Parameter(param[s].view(shape)) for s, shape in zip(carved, shapes)]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        opt = fo.FlashMuon(params, lr=_LR, momentum=_MOMENTUM, weight_decay=_DECAY, quantize=case["quantize"], master_weight_bits=case["master"] or None)
    for p, s, shape in zip(params, carved, shapes):
        p.grad = grad[s].view(shape)
        holder = _MaybeQuantizedTensor(None, try_quantize=case["quantize"], signed=True, sqrt=False, softsign=True, storage_dtype=dtype)
        if case["quantize"]:
            groups = slice(s.start // _GROUP, -(-s.stop // _GROUP))
            holder.load_state_dict({"x::quantized": state["codes"][s].view(shape), "x::scales": state["scales"][groups]}, "x")
        else:
            holder.load_state_dict({"x": state["momentum"][s].view(shape)}, "x")
        opt.state[p]["momentum_buffer"] = holder
        if ecc:
            opt.state[p]["error_bits"] = state["ecc"][s].view(shape)
    state["opt"] = opt


# ------------------------------------------------------------------------------------------------- plain forms


def _iterate(x, steps=_STEPS):
    """The Newton-Schulz iteration on a stack of matrices of the type that `x` has."""
    a, b, c = _COEFFICIENTS
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x.contiguous()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + _NORM_EPS)
    for _ in range(steps):
        gram = torch.bmm(x, x.transpose(1, 2))
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2) if tall else x


def _mx_parts(x):
    """Rows of fp32 values as E2M1 values and one power of two for 32 of them (its exponent); rows are filled up with zeros
    to whole blocks of 128."""
    rows, cols = x.shape
    full = x.new_zeros(rows, -(-cols // 128) * 128)
    full[:, :cols] = x
    groups = full.view(rows, -1, _GROUP)
    largest = groups.abs().amax(2)
    exponent = torch.frexp(largest)[1] - 3
    exponent = torch.where(largest > 0, exponent, -127).clamp(min=-127)
    y = torch.ldexp(groups, -exponent.unsqueeze(2))
    size = y.abs()
    unit = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    near = (torch.round(size / unit) * unit).clamp(max=6.0)
    return torch.copysign(near, y).view(rows, -1), exponent


def _mx_values(x):
    """`x` as its MXFP4 form has it, in fp32."""
    values, exponent = _mx_parts(x.float())
    spread = torch.ldexp(values.view(x.shape[0], -1, _GROUP), exponent.unsqueeze(2))
    return spread.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _mx_unpack(codes, scales, cols):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    values = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], 2).view(codes.shape[0], -1, _GROUP)
    return torch.ldexp(values, scales.int().unsqueeze(2) - 127).view(codes.shape[0], -1)[:, :cols]


def _grouped(x):
    return x.view(-1, _GROUP)


def _moment_codes(m):
    """Codes and fp16 group scales of a momentum whose length is a multiple of the group."""
    groups = _grouped(m)
    scale = groups.abs().amax(1, keepdim=True).clamp(min=1e-12)
    n = groups / scale
    codes = torch.floor((2.0 * n) / (1.0 + n.abs()) * 127.0 + 0.5)
    return codes.to(torch.int8).view(-1), scale.to(torch.float16).view(-1)


def _moment_values(codes, scales):
    y = _grouped(codes.float()) / 127.0
    return (y / (2.0 - y.abs()) * scales.float().unsqueeze(1)).view(-1)


def _half_unit(x):
    """Half of the last place of 16-bit values, in fp32: the correction bits count fractions of it."""
    bits, low = (7, -126) if x.dtype == torch.bfloat16 else (10, -14)
    exponent = torch.frexp(x.float())[1] - 1
    exponent = torch.where(x == 0, low, exponent).clamp(min=low)
    return torch.ldexp(torch.ones((), device="cuda"), exponent - bits - 1)


def _plain_muon(state):
    case = state["case"]
    ecc_top = {0: None, 1: 127.0, 2: 32767.0}[_ecc_bytes(case)]
    grad, param = state["grad"].float(), state["param"]
    keep = float(torch.tensor(1.0) - torch.tensor(_MOMENTUM))
    old = _moment_values(state["codes"], state["scales"]) if case["quantize"] else state["momentum"].float()
    momentum = old * _MOMENTUM + grad * keep
    update = grad * keep + momentum * _MOMENTUM
    master = param.float()
    if ecc_top:
        master = master + state["ecc"].float() / ecc_top * _half_unit(param)
    for at, (r, c) in zip(state["starts"], state["shapes"]):
        s = slice(at, at + r * c)
        step = _iterate(update[s].view(1, r, c)).reshape(-1)
        master[s] = master[s] * (1.0 - _LR * _DECAY) - step * (_LR * math.sqrt(max(1.0, r / c)))
    param.copy_(master)
    if ecc_top:
        state["ecc"].copy_(torch.round(((master - param.float()) / _half_unit(param)).clamp(-1.0, 1.0) * ecc_top))
        master = param.float() + state["ecc"].float() / ecc_top * _half_unit(param)
    if case["quantize"]:
        codes, scales = _moment_codes(momentum)
        state["codes"].copy_(codes)
        state["scales"].copy_(scales)
        momentum = _moment_values(codes, scales)
    else:
        momentum = state["momentum"].copy_(momentum)
    return dict(param=param, master=master, momentum=momentum)


def _plain(state):
    task = state["case"]["task"]
    if task == "ns":
        return _iterate(state["x"].float()).to(torch.bfloat16)
    if task == "muon":
        return _plain_muon(state)
    x = state["x"]
    if task == "quant":
        along, out = state["case"]["along"], {}
        if along != "columns":
            out["rows"] = _mx_values(x).to(torch.bfloat16)
        if along != "rows":
            out["columns"] = _mx_values(x.t()).to(torch.bfloat16)
        return out
    if task == "serve":
        weight = _mx_unpack(state["codes"], state["scales"], x.shape[1])
        return (_mx_values(x) @ weight.t()).to(x.dtype)
    w, dy = state["weight"], state["dy"]
    return dict(
        y=(_mx_values(x) @ _mx_values(w).t()).to(x.dtype),
        dx=(_mx_values(dy) @ _mx_values(w.t()).t()).to(x.dtype),
        dw=(_mx_values(dy.t()) @ _mx_values(x.t()).t()).to(w.dtype))


# ------------------------------------------------------------------------------------------------- one pass


def run(state):
    if not own:
        return _plain(state)
    import flashoptim_amd as fo

    task = state["case"]["task"]
    if task == "ns":
        return fo.newton_schulz(state["x"], steps=_STEPS, coefficients=_COEFFICIENTS, eps=_NORM_EPS)
    if task == "muon":
        state["opt"].step()
        # the weights as an evaluation takes them, and the momentum as a checkpoint holds it
        quantized, param = state["case"]["quantize"], state["param"]
        master = fo.reconstruct_fp32_param(param, state["ecc"]) if "ecc" in state else param
        return dict(param=param, master=master, momentum=_read_momentum(state) if quantized else state["momentum"])
    x = state["x"]
    if task == "quant":
        along = state["case"]["along"]
        if along == "both":
            rows, columns = fo.mxfp4_quantize_both(x)
            return dict(rows=fo.mxfp4_dequantize(rows), columns=fo.mxfp4_dequantize(columns))
        return {along: fo.mxfp4_dequantize(fo.mxfp4_quantize(x, transpose=along == "columns"))}
    if task == "serve":
        weight = fo.MXFP4Tensor(state["codes"], state["scales"], (state["case"]["outer"], state["case"]["inner"]))
        return fo.mxfp4_linear(x, weight)
    leaf, weight = x.detach().requires_grad_(), state["weight"].detach().requires_grad_()
    y = fo.mxfp4_linear(leaf, weight)
    dx, dw = torch.autograd.grad(y, (leaf, weight), state["dy"])
    return dict(y=y.detach(), dx=dx, dw=dw)


def _read_momentum(state):
    from flashoptim_amd.kernels import dequantize

    return dequantize(state["codes"], state["scales"])


# ------------------------------------------------------------------------------------------------- its cost and its exact values


def _iteration_flops(rows, cols):
    """Both Gram products are symmetric, one half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return _STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    width, task = _WIDTH[case["dtype"]], case["task"]
    if task == "ns":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": n * (width + 2), "flops": case["batch"] * _iteration_flops(case["rows"], case["cols"])}
    if task == "muon":
        shapes = _muon_shapes(case)
        n = sum(r * c for r, c in shapes)
        held = 1.0 + 2.0 / _GROUP if case["quantize"] else width
        # gradient in, weight, correction bits and momentum in and out; the masters and the momentum read once more and
        # handed out in fp32
        per = 3 * width + 2 * _ecc_bytes(case) + 2 * held
        per += (width + _ecc_bytes(case) + 4 if _ecc_bytes(case) else 0) + (held + 4 if case["quantize"] else 0)
        return {"bytes": n * per, "flops": sum(_iteration_flops(r, c) for r, c in shapes) + 30 * n}
    packed = 17.0 / 32.0
    if task == "quant":
        n, forms = case["rows"] * case["cols"], 2 if case["along"] == "both" else 1
        return {"bytes": n * (width + forms * (2 * packed + 2)), "flops": 6 * forms * n}
    t, k, n = case["tokens"], case["inner"], case["outer"]
    if task == "serve":
        return {"bytes": n * k * packed + t * (k + n) * width, "flops": 2 * t * k * n}
    # inputs and gradients once each; both forms of the three operands written and read
    return {"bytes": width * 2 * (t * k + n * k) + width * 2 * t * n + 4 * packed * (t * k + n * k + t * n), "flops": 6 * t * k * n}


def exact(case, seed):
    """Definitions in 64 bits.  Codes are decided on the inputs, which are the same numbers in 64 bits."""
    import types

    if case["task"] == "muon":
        # before prepare()'s optimizer, which this does not need
        state, g = dict(case=case), torch.Generator(device="cuda").manual_seed(seed)
        keep, here = globals()["own"], globals()
        here["own"] = False
        try:
            _prepare_muon(state, case, g, _DTYPES[case["dtype"]])
        finally:
            here["own"] = keep
        return _exact_muon(types.SimpleNamespace(**state))
    state = prepare(case, seed)
    if case["task"] == "ns":
        return _exact_polynomial(state["x"].double())
    x = state["x"].double()
    if case["task"] == "quant":
        both = {"rows": lambda: _exact_mx(x), "columns": lambda: _exact_mx(x.t())}
        return {k: f() for k, f in both.items() if case["along"] in (k, "both")}
    if case["task"] == "serve":
        low, high = state["codes"].long() & 15, state["codes"].long() >> 4
        code = torch.stack((low, high), -1).flatten(1)
        fraction, power = (code & 1).double(), (code >> 1) & 3
        size = torch.where(power > 0, (1 + fraction / 2) * torch.exp2((power - 1).double()), fraction / 2)
        weight = torch.where(code > 7, -size, size) * torch.exp2(state["scales"].double() - 127).repeat_interleave(_GROUP, 1)
        return torch.mm(_exact_mx(x), weight[:, :x.shape[1]].t().contiguous())
    w, dy = state["weight"].double(), state["dy"].double()
    return {
        "y": torch.mm(_exact_mx(x), _exact_mx(w).t()),
        "dx": torch.mm(_exact_mx(dy), _exact_mx(w.t()).t()),
        "dw": torch.mm(_exact_mx(dy.t()), _exact_mx(x.t()).t())}


def _exact_mx(x):
    """The nearest of the eight magnitudes by search, even codes at ties, times the group's power of two."""
    rows, cols = x.shape
    groups = torch.nn.functional.pad(x, (0, -cols % _GROUP)).unflatten(1, (-1, _GROUP))
    power = torch.exp2(torch.floor(torch.log2(groups.abs().amax(-1, keepdim=True))).clamp(min=-125) - 2)
    # values halfway go to the even code: the borders between neighbours belong to the even one of the two
    size = (groups / power).abs()
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    code = torch.zeros_like(size)
    for i in range(7):
        border = (grid[i] + grid[i + 1]) / 2
        code += (size > border) | ((size == border) & (i % 2 == 1))
    return (grid[code.long()] * groups.sign() * power).flatten(1)[:, :cols]


def _exact_polynomial(x):
    """X <- p(X X') X with p(t) = a + b t + c t^2, on the shorter side, in 64 bits."""
    a, b, c = _COEFFICIENTS
    out = []
    for matrix in x:
        wide = matrix if matrix.shape[0] <= matrix.shape[1] else matrix.t()
        z = wide / (torch.linalg.norm(wide) + _NORM_EPS)
        eye = torch.eye(z.shape[0], dtype=z.dtype, device=z.device)
        for _ in range(_STEPS):
            s = z @ z.t()
            z = (a * eye + s @ (b * eye + c * s)) @ z
        out.append(z if wide is matrix else z.t())
    return torch.stack(out)


def _exact_muon(s):
    ecc = _ecc_bytes(s.case)
    keep = float(torch.tensor(1.0) - torch.tensor(_MOMENTUM))
    mu = float(torch.tensor(_MOMENTUM))
    grad = s.grad.double()
    if s.case["quantize"]:
        y = s.codes.double() / 127
        old = y / (2 - y.abs()) * s.scales.double().repeat_interleave(_GROUP)
    else:
        old = s.momentum.double()
    new = mu * old + keep * grad
    direction = keep * grad + mu * new
    master = s.param.double()
    if ecc:
        bits, low = (7, -126) if s.param.dtype == torch.bfloat16 else (10, -14)
        exponent = torch.floor(torch.log2(master.abs())).clamp(min=low)
        master = master + s.ecc.double() / (127 if ecc == 1 else 32767) * torch.exp2(exponent - bits - 1)
    for at, (r, c) in zip(s.starts, s.shapes):
        part = slice(at, at + r * c)
        step = _exact_polynomial(direction[part].view(1, r, c)).flatten()
        master[part] = master[part] * (1 - _LR * _DECAY) - _LR * max(1.0, r / c) ** 0.5 * step
    if s.case["quantize"]:
        groups = new.unflatten(0, (-1, _GROUP))
        top = groups.abs().amax(1, keepdim=True).clamp(min=1e-12)
        code = torch.floor(2 * groups / (top + groups.abs()) * 127 + 0.5) / 127
        new = (code / (2 - code.abs()) * top.to(torch.float16).double()).flatten()
    # the weight is the master rounded to its type
    return {"param": master, "master": master, "momentum": new}
