"""The two ends of a language model and the joints between its layers, as timed cases.

What stands before, between and after the linear layers of a model that this package trains and serves:

* ``embed``  tokens to rows of an embedding matrix, scaled, and the matrix's gradient;
* ``norm``   the residual stream's addition with the root-mean-square norm that follows it, and their gradients; for serving the
             norm's output goes into MXFP4, which the layers' products read;
* ``loss``   hidden states to the cross entropy over a vocabulary, through the output matrix, without the logits in memory, and
             the gradients of both.

A case is one call of one of them, with its backward pass where ``train`` is set.  Tokens follow a Zipf distribution over a
shuffled vocabulary, a share of them may be one padding token; of the hidden states some predict their target nearly surely and
some not at all.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_WIDTH = {"bf16": 2, "fp16": 2, "fp32": 4}
_GROUP = 32        # values of an MXFP4 row that share one scale
_EPS = 1e-5
_IGNORE = -100


# ------------------------------------------------------------------------------------------------- the cases


def _embed(name, dtype, tokens, vocabulary, width, scale=1.0, padding=0.0, index="int64", train=True):
    return dict(name=name, task="embed", dtype=dtype, tokens=tokens, vocabulary=vocabulary, width=width, scale=scale, padding=padding, index=index,
                train=train)


def _norm(name, dtype, stream, tokens, width, train=True, mxfp4=False, margin=0):
    """stream: the residual's type, or "none"; margin: columns of the wider matrix that the input is a part of."""
    return dict(name=name, task="norm", dtype=dtype, stream=stream, tokens=tokens, width=width, train=train, mxfp4=mxfp4, margin=margin)


def _loss(name, dtype, tokens, width, vocabulary, reduction="mean", smoothing=0.0, ignored=0.0, train=True):
    return dict(name=name, task="loss", dtype=dtype, tokens=tokens, width=width, vocabulary=vocabulary, reduction=reduction, smoothing=smoothing,
                ignored=ignored, train=train)


def listed():
    return [
        # a training batch into the 8B-parameter transformer that the package's benchmark steps, and its matrix's gradient
        _embed("embed-8b", "bf16", 8192, 128256, 4096),
        # a padded batch of a small model with odd widths, embeddings scaled by the root of the width
        _embed("embed-odd", "fp32", 1003, 5003, 250, math.sqrt(250.0), 0.3),
        # one token of an answer
        _embed("embed-one", "bf16", 1, 128256, 4096, train=False),
        # a joint of that transformer over a training batch
        _norm("norm-8b", "bf16", "bf16", 8192, 4096),
        # the same of a small model in fp16 that keeps its residual stream in fp32; the input is a part of a wider product
        _norm("norm-odd", "fp16", "fp32", 1003, 2730, margin=24),
        # a prompt on its way into MXFP4 layers
        _norm("norm-prompt", "bf16", "bf16", 4096, 4096, train=False, mxfp4=True),
        # one token of an answer, the same
        _norm("norm-one", "bf16", "bf16", 1, 4096, train=False, mxfp4=True),
        # the transformer's loss over a training batch
        _loss("loss-8b", "bf16", 8192, 4096, 128256),
        # fine-tuning a small model with odd sizes on a masked batch
        _loss("loss-odd", "fp16", 1003, 1000, 32003, "sum", 0.1, 0.4),
        # the example's language model: few words, many tokens
        _loss("loss-words", "bf16", 4096, 512, 64),
        # a small model whose ends stay in fp32
        _loss("loss-fp32", "fp32", 512, 1000, 5003, "none", 0.0, 0.1),
        # log-probabilities of a few drafted tokens
        _loss("loss-score", "bf16", 5, 4096, 128256, "none", train=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(2 ** rng.uniform(math.log2(lo), math.log2(hi))))

    task = rng.choice(["embed", "norm", "norm", "loss", "loss", "loss"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.75
    if task == "embed":
        while True:
            tokens, vocabulary, width = log(1, 65536), log(64, 128256), log(32, 8192)
            if (tokens + vocabulary) * width * _WIDTH[dtype] <= 128256 * 4096 * 2:
                break
        case = _embed("", dtype, tokens, vocabulary, width, rng.choice([1.0, math.sqrt(width)]), rng.choice([0.0, 0.0, 0.3, 0.9]),
                      rng.choice(["int64", "int64", "int32"]), train)
    elif task == "norm":
        while True:
            tokens, width = log(1, 16384), log(32, 16384)
            if tokens * width <= 8192 * 4096:
                break
        stream = rng.choice([dtype, dtype, "fp32", "none"])
        case = _norm("", dtype, stream, tokens, width, train, not train and rng.random() < 0.5, rng.choice([0, 0, 24]))
    else:
        while True:
            tokens, width, vocabulary = log(1, 8192), log(32, 4096), log(64, 128256)
            if tokens * width * vocabulary <= 8192 * 4096 * 128256 / (8 if dtype == "fp32" else 1):
                break
        case = _loss("", dtype, tokens, width, vocabulary, rng.choice(["mean", "mean", "sum", "none"]), rng.choice([0.0, 0.0, 0.1]),
                     rng.choice([0.0, 0.1, 0.9]), train)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------- inputs


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _zipf(g, n, vocabulary):
    """n tokens, the k-th most frequent about 1 / (k + 2) as frequent as the first."""
    rank = (2.0 * (vocabulary / 2.0 + 1.0) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64) - 2.0).long().clamp_(0, vocabulary - 1)
    return torch.randperm(vocabulary, generator=g, device="cuda")[rank]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, n, d = _DTYPES[case["dtype"]], case["tokens"], case["width"]
    state = dict(case=case)
    if case["task"] == "embed":
        v = case["vocabulary"]
        tokens = _zipf(g, n, v)
        state["padding"] = v - 1 if case["padding"] else None
        tokens[torch.rand(n, generator=g, device="cuda") < case["padding"]] = v - 1
        state["tokens"] = tokens.to(getattr(torch, case["index"]))
        state["weight"] = _normal(g, v, d).mul_(0.02).to(dtype)
        if case["train"]:
            state["dy"] = _normal(g, n, d).mul_(1e-3).to(dtype)
    elif case["task"] == "norm":
        more = case["margin"]
        # some channels far larger than the rest, as in the middle of a deep model
        large = 1.0 + 7.0 * (torch.rand(d, generator=g, device="cuda") < 0.01)
        state["x"] = _normal(g, n, d + more).to(dtype)[:, more // 2:more // 2 + d]
        state["weight"] = (1.0 + 0.1 * _normal(g, d)).to(dtype)
        state["residual"] = None if case["stream"] == "none" else (3.0 * _normal(g, n, d) * large).to(_DTYPES[case["stream"]])
        if case["train"]:
            state["dy"] = (1e-3 * _normal(g, n, d)).to(dtype)
            state["dstream"] = None if case["stream"] == "none" else (1e-3 * _normal(g, n, d)).to(_DTYPES[case["stream"]])
    else:
        v = case["vocabulary"]
        weight = _normal(g, v, d).mul_(1.3 / math.sqrt(d))
        target = _zipf(g, n, v)
        # what the hidden state knows of its target: from nothing to a logit of 15 above the others
        known = torch.rand(n, 1, generator=g, device="cuda") * (8.0 * torch.randint(0, 2, (n, 1), generator=g, device="cuda"))
        state["x"] = (_normal(g, n, d) + known * weight[target]).to(dtype)
        state["weight"] = weight.to(dtype)
        if case["ignored"]:
            ignored = torch.rand(n, generator=g, device="cuda") < case["ignored"]
            ignored[0] = False
            target[ignored] = _IGNORE
        state["target"] = target
        if case["train"]:  # what a loss is multiplied by on its way back
            state["upstream"] = torch.rand(n, generator=g, device="cuda") / n if case["reduction"] == "none" else torch.ones((), device="cuda")
    return state


# ------------------------------------------------------------------------------------------------- plain forms


def _plain_embed(state):
    case, weight, tokens = state["case"], state["weight"], state["tokens"].long()
    y = (weight[tokens].float() * case["scale"]).to(weight.dtype)
    if not case["train"]:
        return y
    dy = state["dy"].float() * case["scale"]
    if state["padding"] is not None:
        dy = dy * (tokens != state["padding"]).unsqueeze(1)
    dw = torch.zeros(weight.shape, device="cuda").index_add_(0, tokens, dy)
    return dict(y=y, dw=dw.to(weight.dtype))


def _mx_values(x):
    """fp32 rows as MXFP4 has them: E2M1 values times one power of two for each 32."""
    rows, cols = x.shape
    full = x.new_zeros(rows, -(-cols // _GROUP) * _GROUP)
    full[:, :cols] = x
    groups = full.view(rows, -1, _GROUP)
    largest = groups.abs().amax(2)
    exponent = torch.where(largest > 0, torch.frexp(largest)[1] - 3, -127).clamp(min=-127).unsqueeze(2)
    y = torch.ldexp(groups, -exponent)
    size = y.abs()
    unit = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    near = (torch.round(size / unit) * unit).clamp(max=6.0)
    return torch.ldexp(torch.copysign(near, y), exponent).view(rows, -1)[:, :cols]


def _plain_norm(state):
    case, residual = state["case"], state["residual"]
    x, w = state["x"].float(), state["weight"].float()
    stream = None
    if residual is not None:
        stream = (x + residual.float()).to(residual.dtype)
        x = stream.float()
    inverse = torch.rsqrt(x.square().mean(1, keepdim=True) + _EPS)
    n = x * inverse
    out = {} if stream is None else dict(stream=stream)
    if case["mxfp4"]:
        return dict(out, y=_mx_values(n * w).to(torch.bfloat16))
    out["y"] = (n * w).to(state["x"].dtype)
    if not case["train"]:
        return out
    dy = state["dy"].float()
    dn = dy * w
    dx = inverse * (dn - n * (dn * n).mean(1, keepdim=True))
    if stream is not None:
        dx = dx + state["dstream"].float()
        out["dresidual"] = dx.to(residual.dtype)
    return dict(out, dx=dx.to(state["x"].dtype), dw=(dy * n).sum(0).to(state["weight"].dtype))


def _plain_loss(state):
    case, target = state["case"], state["target"]
    x, w = state["x"].float(), state["weight"].float()
    smoothing, v = case["smoothing"], case["vocabulary"]
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    total = (logits - top).exp().sum(1, keepdim=True)
    lse = total.log() + top
    kept = target != _IGNORE
    at = torch.where(kept, target, 0).unsqueeze(1)
    loss = lse - (1.0 - smoothing) * logits.gather(1, at)
    if smoothing:
        loss = loss - smoothing * logits.mean(1, keepdim=True)
    loss = loss.squeeze(1) * kept
    count = kept.sum()
    out = dict(loss=loss if case["reduction"] == "none" else loss.sum() if case["reduction"] == "sum" else loss.sum() / count)
    if not case["train"]:
        return out
    factor = kept * state["upstream"]
    if case["reduction"] == "mean":
        factor = factor / count
    grad = logits.sub_(lse).exp_()
    if smoothing:
        grad.sub_(smoothing / v)
    grad.scatter_add_(1, at, torch.full_like(lse, smoothing - 1.0))
    grad.mul_(factor.unsqueeze(1))
    return dict(out, dx=(grad @ w).to(state["x"].dtype), dw=(grad.t() @ x).to(state["weight"].dtype))


# ------------------------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if not own:
        return dict(embed=_plain_embed, norm=_plain_norm, loss=_plain_loss)[case["task"]](state)
    import flashoptim_amd as fo

    if case["task"] == "embed":
        if not case["train"]:
            return fo.embedding(state["tokens"], state["weight"], scale=case["scale"])
        weight = state["weight"].detach().requires_grad_()
        y = fo.embedding(state["tokens"], weight, scale=case["scale"], padding_idx=state["padding"])
        return dict(y=y.detach(), dw=torch.autograd.grad(y, weight, state["dy"])[0])
    if case["task"] == "norm":
        x, weight, residual = state["x"], state["weight"], state["residual"]
        if case["mxfp4"]:
            got = fo.rms_norm_mxfp4(x, weight, residual, eps=_EPS)
            y, stream = (got, None) if residual is None else got
            return dict({} if stream is None else dict(stream=stream), y=y.dequantize(torch.bfloat16))
        if not case["train"]:
            got = fo.rms_norm(x, weight, residual, eps=_EPS)
            return dict(y=got) if residual is None else dict(stream=got[1], y=got[0])
        leaves = [t.detach().requires_grad_() for t in (x, weight, residual) if t is not None]
        if residual is None:
            y = fo.rms_norm(*leaves, eps=_EPS)
            dx, dw = torch.autograd.grad(y, leaves, state["dy"])
            return dict(y=y.detach(), dx=dx, dw=dw)
        y, stream = fo.rms_norm(*leaves, eps=_EPS)
        dx, dw, dresidual = torch.autograd.grad((y, stream), leaves, (state["dy"], state["dstream"]))
        return dict(stream=stream.detach(), y=y.detach(), dresidual=dresidual, dx=dx, dw=dw)
    how = dict(ignore_index=_IGNORE, reduction=case["reduction"], label_smoothing=case["smoothing"])
    if not case["train"]:
        return dict(loss=fo.linear_cross_entropy(state["x"], state["weight"], state["target"], **how))
    x, weight = state["x"].detach().requires_grad_(), state["weight"].detach().requires_grad_()
    loss = fo.linear_cross_entropy(x, weight, state["target"], **how)
    dx, dw = torch.autograd.grad(loss, (x, weight), state["upstream"])
    return dict(loss=loss.detach(), dx=dx, dw=dw)


# ------------------------------------------------------------------------------------------------- its cost and its exact values


def work(case):
    width, n, d = _WIDTH[case["dtype"]], case["tokens"], case["width"]
    if case["task"] == "embed":
        v, index = case["vocabulary"], 8 if case["index"] == "int64" else 4
        moved = n * index + (min(n, v) + n) * d * width
        return {"bytes": moved + ((n + v) * d * width if case["train"] else 0), "flops": n * d * (2 if case["train"] else 1)}
    if case["task"] == "norm":
        stream = _WIDTH.get(case["stream"], 0)
        out = 2 + 2 * 17.0 / 32.0 if case["mxfp4"] else width    # codes written, read and handed out as bf16
        per = width + out + 2 * stream
        if case["train"]:
            per += 2 * width + 2 * stream    # dy in, dx out; the stream's gradient in and out
        return {"bytes": n * d * per + d * width, "flops": n * d * (16 if case["train"] else 6)}
    v, train = case["vocabulary"], case["train"]
    moved = (n + v) * d * width * (2 if train else 1) + n * 8
    return {"bytes": moved, "flops": (6 if train else 2) * n * d * v}


def exact(case, seed):
    """Definitions in 64 bits."""
    state = prepare(case, seed)
    return {"embed": _exact_embed, "norm": _exact_norm, "loss": _exact_loss}[case["task"]](case, state)


def _exact_embed(case, s):
    rows = torch.index_select(s["weight"], 0, s["tokens"].reshape(-1)).double() * case["scale"]
    if not case["train"]:
        return rows
    # tokens in order, sums of their runs by differences of a running sum of each row's share
    order = torch.argsort(s["tokens"].long(), stable=True)
    sorted_tokens = s["tokens"].long()[order]
    first, count = torch.unique_consecutive(sorted_tokens, return_counts=True)
    ends = count.cumsum(0)
    running = torch.nn.functional.pad(s["dy"].double()[order].cumsum(0), (0, 0, 1, 0))
    dw = torch.zeros(s["weight"].shape, dtype=torch.float64, device="cuda")
    dw[first] = (running[ends] - running[ends - count]) * case["scale"]
    if s["padding"] is not None:
        dw[s["padding"]] = 0
    return {"y": rows, "dw": dw}


def _exact_norm(case, s):
    z = s["x"].double()
    out = {}
    if s["residual"] is not None:
        # the stream is what is kept of the sum, and what the norm reads
        out["stream"] = z + s["residual"].double()
        z = out["stream"].to(s["residual"].dtype).double()
    size = (torch.linalg.vector_norm(z, dim=1, keepdim=True) ** 2 / z.shape[1] + _EPS) ** 0.5
    w = s["weight"].double()
    y = z / size * w
    if case["mxfp4"]:
        return {**out, "y": _exact_mx(y)}
    out["y"] = y
    if not case["train"]:
        return out
    dy = s["dy"].double()
    # y_j = w_j z_j / size;  d size / d z_i = z_i / (d size)
    along = (dy * y).sum(1, keepdim=True)
    dx = dy * w / size - z * along / (z.shape[1] * size ** 2)
    out_dw = torch.mv((dy * (z / size)).t().contiguous(), torch.ones(z.shape[0], dtype=torch.float64, device="cuda"))
    if s["residual"] is None:
        return {**out, "dx": dx, "dw": out_dw}
    dx = dx + s["dstream"].double()
    return {**out, "dresidual": dx, "dx": dx, "dw": out_dw}


def _exact_mx(x):
    """The nearest of the eight magnitudes by search, even codes at ties, times the group's power of two."""
    cols = x.shape[1]
    groups = torch.nn.functional.pad(x, (0, -cols % _GROUP)).unflatten(1, (-1, _GROUP))
    power = torch.exp2(torch.floor(torch.log2(groups.abs().amax(-1, keepdim=True))).clamp(min=-125) - 2)
    size = (groups / power).abs()
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    code = sum(((size > (grid[i] + grid[i + 1]) / 2) | ((size == (grid[i] + grid[i + 1]) / 2) & (i % 2 == 1))).long() for i in range(7))
    return (grid[code] * groups.sign() * power).flatten(1)[:, :cols]


def _exact_loss(case, s):
    x, w, target = s["x"].double(), s["weight"].double(), s["target"]
    v, e = w.shape[0], case["smoothing"]
    logp = torch.nn.functional.log_softmax(torch.mm(x, w.t()), 1)
    live = torch.nonzero(target != _IGNORE).squeeze(1)
    wanted = target[live]
    each = torch.zeros(x.shape[0], dtype=torch.float64, device="cuda")
    each[live] = -(1 - e) * logp[live, wanted] - (e * logp.mean(1)[live] if e else 0)
    out = {"loss": {"none": lambda: each, "sum": each.sum, "mean": lambda: each.sum() / live.numel()}[case["reduction"]]()}
    if not case["train"]:
        return out
    share = torch.zeros(x.shape[0], dtype=torch.float64, device="cuda")
    share[live] = s["upstream"].double()[live] if case["reduction"] == "none" else s["upstream"].double() / (live.numel() if case["reduction"] == "mean" else 1)
    p = logp.exp_()
    p -= e / v
    p[live, wanted] -= 1 - e
    p *= share[:, None]
    return {**out, "dx": torch.mm(p, w), "dw": torch.mm(p.t(), x)}
