"""The head, the teacher's targets and the distillation loss as timed cases, each beside a plain form.

Four kinds of case:

``top``         ``top_logits(logits, k, temperature)``: a teacher's k largest logits of each row, their
                classes, and the log of what all other classes sum to.
``distill``     ``distill_loss`` through autograd: the loss, then the gradient of the student's logits.
``distill_one`` ``distill_loss_grad``: loss and gradient of the student's logits in one call.
``linear``      ``linear_act`` under ``no_grad``: product, bias, activation and residual.
``linear_train`` the same through autograd, with the gradient of every input.

``own`` chooses between the framework's calls and the plain form: elementary float32 operations,
rounded once to the inputs' type at the end.

Ranges (``draw``): 1 to 8192 rows of logits over 100 to 150000 classes, 1 to 128 teacher entries a row,
some rows without any; products of 1 to 100352 rows with 16 to 8192 inputs and outputs; float32 (logits),
float16 and bfloat16.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}

# Bounds of drawn cases: what the largest listed ones of a kind have.
_MOST_TOP = 4096 * 32768
_MOST_LOGIT_BYTES = 4096 * 128000 * 2
_MOST_FLOPS = 6 * 8192 * 2048 * 8192
_MOST_ELEMENTS = 8192 * 8192


def _top(dtype, rows, classes, k, t=1.0):
    return {"kind": "top", "dtype": dtype, "rows": rows, "classes": classes, "k": k, "t": t}


def _distill(kind, dtype, rows, classes, k, t=2.0, rest=True, reduction="mean"):
    return {"kind": kind, "dtype": dtype, "rows": rows, "classes": classes, "k": k, "t": t, "rest": rest,
            "reduction": reduction}


def _linear(kind, dtype, rows, inputs, outputs, act="none", bias=True, residual="none"):
    return {"kind": kind, "dtype": dtype, "rows": rows, "inputs": inputs, "outputs": outputs, "act": act,
            "bias": bias, "residual": residual}


def listed():
    return [
        # The teacher's targets for an ImageNet batch: a call of a few microseconds inside the training loop.
        {"name": "top_imagenet_batch", **_top("f16", 256, 1000, 20, 2.0)},
        # Targets over a vocabulary, for a batch of token sequences.
        {"name": "top_vocabulary", **_top("bf16", 4096, 32768, 64)},
        # A class count and a k that nothing divides, float32, few rows.
        {"name": "top_odd_f32", **_top("f32", 77, 50021, 33, 4.0)},
        # One ImageNet batch of distillation under mixed precision.
        {"name": "distill_imagenet", **_distill("distill", "f16", 256, 1000, 20)},
        # The loss over a large vocabulary, loss and gradient in one call as a chunked head takes them.
        {"name": "distill_vocabulary", **_distill("distill_one", "bf16", 4096, 128000, 64)},
        # float32 logits over an odd class count, only the top classes as targets, a weight for each row.
        {"name": "distill_odd_f32", **_distill("distill", "f32", 1031, 32003, 17, 1.0, False, "none")},
        # The classifier on one image: a call's latency.
        {"name": "linear_one_row", **_linear("linear", "f16", 1, 2048, 1000)},
        # Thirty-two sequences, one token each, through a hidden layer.
        {"name": "linear_few_rows", **_linear("linear", "bf16", 32, 4096, 4096, "silu")},
        # The third 1x1 convolution of a second-stage bottleneck on 128 images, channels_last: bias, shortcut, ReLU.
        {"name": "linear_expand_pixels", **_linear("linear", "f16", 128 * 28 * 28, 128, 512, "relu", True, "before")},
        # The classifier's training step at an ImageNet batch.
        {"name": "linear_train_classifier", **_linear("linear_train", "f16", 256, 2048, 1000)},
        # Sizes that no tile divides.
        {"name": "linear_train_odd", **_linear("linear_train", "bf16", 1001, 577, 1003, "silu", True, "after")},
        # A hidden layer's training step on 8192 tokens.
        {"name": "linear_train_large", **_linear("linear_train", "bf16", 8192, 2048, 8192, "gelu")},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    """A layer's width: mostly as networks have them, a third of any number."""
    if rng.random() < 0.33:
        return _log_int(rng, 16, 8192)
    return rng.choice([64, 96, 128, 256, 512, 768, 1000, 1024, 2048, 4096, 8192])


def draw(rng):
    kind = rng.choice(["top", "distill", "distill_one", "linear", "linear_train"])
    if kind in ("top", "distill", "distill_one"):
        dtype = rng.choice(["f32", "f16", "bf16"])
        classes = rng.choice([1000, 21841, 32000, 65536, 128000]) if rng.random() < 0.4 else _log_int(rng, 100, 150000)
        most = _MOST_TOP if kind == "top" else _MOST_LOGIT_BYTES // _BYTES[dtype]
        rows = max(1, min(_log_int(rng, 1, 8192), most // classes))
        k, t = _log_int(rng, 1, min(128, classes // 2)), rng.choice([1.0, 2.0, 4.0])
        if kind == "top":
            return _top(dtype, rows, classes, k, t)
        return _distill(kind, dtype, rows, classes, k, t, rng.random() < 0.6, rng.choice(["mean", "none", "sum"]))
    inputs, outputs = _width(rng), _width(rng)
    rows = _log_int(rng, 1, 128 * 28 * 28)
    flops = (2 if kind == "linear" else 6) * inputs * outputs
    rows = max(1, min(rows, _MOST_FLOPS // flops, _MOST_ELEMENTS // max(inputs, outputs)))
    return _linear(kind, rng.choice(["f16", "bf16"]), rows, inputs, outputs,
                   rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.8,
                   rng.choice(["none", "before", "after"]))


def _teacher_logits(case, g):
    """Logits of a trained classifier: a broad floor, and a few classes well above it."""
    n, v = case["rows"], case["classes"]
    x = torch.randn(n, v, generator=g, device="cuda")
    x += torch.randn(n, v, generator=g, device="cuda").sub_(2.5).relu_().mul_(6.0)
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    if case["kind"] == "top":
        return {"case": case, "logits": _teacher_logits(case, g).to(dt)}
    if case["kind"] in ("distill", "distill_one"):
        n, v, t = case["rows"], case["classes"], case["t"]
        x = _teacher_logits(case, g)
        values, indices = x.topk(case["k"], dim=1)
        state = {"case": case, "indices": indices, "rest": None}
        if case["rest"]:
            listed_away = x.scatter(1, indices, float("-inf")).div_(t)
            state["rest"] = listed_away.logsumexp(1)
            del listed_away
        state["values"] = values.to(dt)
        # padding and other rows that are left out
        indices[torch.rand(n, generator=g, device="cuda") < 0.05] = -1
        # the student: near its teacher, not there yet
        x.mul_(0.7).add_(torch.randn(n, v, generator=g, device="cuda"), alpha=0.7)
        state["logits"] = x.to(dt)
        scale = 2.0 ** 14 if case["dtype"] == "f16" else 1.0  # as a loss scaler has it
        state["scale"] = scale
        if case["kind"] == "distill":
            state["logits"].requires_grad_()
            if case["reduction"] == "none":
                state["upstream"] = torch.rand(n, generator=g, device="cuda") * (scale / n)
            else:
                state["upstream"] = torch.tensor(scale if case["reduction"] == "mean" else scale / n, device="cuda")
        return state
    m, k, n = case["rows"], case["inputs"], case["outputs"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    x = normal(m, k)
    if case["act"] == "relu":
        x.relu_()
    state = {"case": case, "x": x.to(dt), "weight": (normal(n, k) / math.sqrt(k)).to(dt),
             "bias": (0.3 * normal(n)).to(dt) if case["bias"] else None,
             "residual": normal(m, n).to(dt) if case["residual"] != "none" else None}
    if case["kind"] == "linear_train":
        for name in ("x", "weight", "bias", "residual"):
            if state[name] is not None:
                state[name].requires_grad_()
        state["upstream"] = normal(m, n).to(dt)
    return state


# ------------------------------------------------------------------ plain forms
def _plain_lse(x):
    """Logarithm of the sum of exponentials of each row; minus infinity for a row of nothing else."""
    m = x.amax(1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    return m[:, 0] + (x - m).exp_().sum(1).log()


def _plain_log_softmax(x):
    """x - lse(x), exact where one entry has nearly everything: the others' sum goes through log1p."""
    m, at = x.max(1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    return (x - m) - (x - m).exp_().scatter_(1, at, 0.0).sum(1, keepdim=True).log1p()


def _plain_without(x, indices):
    """`x` with minus infinity in the listed columns."""
    columns = torch.where((indices >= 0) & (indices < x.shape[1]), indices, x.shape[1])
    wider = torch.cat([x, x.new_empty(x.shape[0], 1)], 1)
    return wider.scatter_(1, columns, float("-inf"))[:, :-1]


def _plain_top(logits, k, t):
    x = logits.float()
    indices = x.sort(dim=1, descending=True, stable=True)[1][:, :k].contiguous()
    return {"values": logits.gather(1, indices), "indices": indices, "rest": _plain_lse(_plain_without(x / t, indices))}


def _plain_distill(logits, values, indices, rest, t, reduction, upstream):
    n, v = logits.shape
    s = logits.float() / t
    there = (indices >= 0) & (indices < v)
    columns = indices.clamp(0, v - 1)
    low = torch.full((n, 1), float("-inf"), device=s.device)
    a = torch.cat([torch.where(there, values.float() / t, low), low if rest is None else rest.float()[:, None]], 1)
    others = _plain_without(s, indices)
    b_rest = _plain_lse(others)
    b = torch.cat([torch.where(there, s.gather(1, columns), low), b_rest[:, None]], 1)
    counted = there.any(1) & (a.amax(1) > float("-inf"))
    log_p, log_q = _plain_log_softmax(a), _plain_log_softmax(b)
    p, q = log_p.exp(), log_q.exp()
    # p log(p/q), written as p log(p/q) - p + q, which sums to the same: no term is negative, nothing cancels
    d = torch.where(p > 0, log_p - log_q, 0.0)
    losses = torch.where(counted, torch.where(p > 0, p * (d + torch.expm1(-d)), q).sum(1) * (t * t), 0.0)
    if reduction == "none":
        loss, each = losses, upstream
    else:
        count = counted.sum().clamp(min=1) if reduction == "mean" else 1
        loss, each = losses.sum() / count, (upstream / count).expand(n)
    each = torch.where(counted, each * t, 0.0)[:, None]
    d = torch.where(p > 0, p * torch.expm1(-d), q) * each  # (q - p) of each bucket
    grad = (others - b_rest[:, None]).exp_().mul_(d[:, -1:])
    grad.scatter_add_(1, columns, torch.where(there, d[:, :-1], 0.0))
    return {"loss": loss, "grad": grad.to(logits.dtype)}


def _plain_act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + (-z).exp())
    return z


def _plain_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * (-0.5 * z * z).exp() / math.sqrt(2 * math.pi)
    if act == "silu":
        s = 1 / (1 + (-z).exp())
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_linear(state):
    case, dt = state["case"], state["x"].dtype
    x, w = state["x"].detach().float(), state["weight"].detach().float()
    z = x @ w.t()
    if state["bias"] is not None:
        z = z + state["bias"].detach().float()
    if case["residual"] == "before":
        z = z + state["residual"].detach().float()
    y = _plain_act(z, case["act"])
    if case["residual"] == "after":
        y = y + state["residual"].detach().float()
    if case["kind"] == "linear":
        return {"y": y.to(dt)}
    gy = state["upstream"].float()
    gz = gy * _plain_slope(z, case["act"])
    out = {"y": y.to(dt), "x": (gz @ w).to(dt), "weight": (gz.t() @ x).to(dt)}
    if state["bias"] is not None:
        out["bias"] = gz.sum(0).to(dt)
    if case["residual"] != "none":
        out["residual"] = (gz if case["residual"] == "before" else gy).to(dt)
    return out


def _plain(state):
    case = state["case"]
    if case["kind"] == "top":
        return _plain_top(state["logits"], case["k"], case["t"])
    if case["kind"] in ("distill", "distill_one"):
        upstream = state["upstream"] if case["kind"] == "distill" else torch.tensor(state["scale"], device="cuda")
        if case["kind"] == "distill_one" and case["reduction"] == "none":
            upstream = upstream.expand(case["rows"])
        return _plain_distill(state["logits"].detach(), state["values"], state["indices"], state["rest"], case["t"],
                              case["reduction"], upstream)
    return _plain_linear(state)


# ------------------------------------------------------------------ the framework's calls
def _own(state):
    from ddfnet_b200 import distill_loss, distill_loss_grad, linear_act, top_logits
    case = state["case"]
    if case["kind"] == "top":
        top = top_logits(state["logits"], case["k"], temperature=case["t"])
        return {"values": top.values, "indices": top.indices, "rest": top.rest}
    if case["kind"] == "distill":
        loss = distill_loss(state["logits"], state["values"], state["indices"], state["rest"],
                            temperature=case["t"], reduction=case["reduction"])
        grad, = torch.autograd.grad(loss, state["logits"], state["upstream"])
        return {"loss": loss, "grad": grad}
    if case["kind"] == "distill_one":
        loss, grad = distill_loss_grad(state["logits"], state["values"], state["indices"], state["rest"],
                                       temperature=case["t"], reduction=case["reduction"], scale=state["scale"])
        return {"loss": loss, "grad": grad}
    add = case["residual"] if case["residual"] != "none" else "before"
    if case["kind"] == "linear":
        with torch.no_grad():
            return {"y": linear_act(state["x"], state["weight"], state["bias"], state["residual"],
                                    activation=case["act"], add=add)}
    y = linear_act(state["x"], state["weight"], state["bias"], state["residual"], activation=case["act"], add=add)
    names = [n for n in ("x", "weight", "bias", "residual") if state[n] is not None]
    return {"y": y, **dict(zip(names, torch.autograd.grad(y, [state[n] for n in names], state["upstream"])))}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    es = _BYTES[case["dtype"]]
    if case["kind"] == "top":
        n, v, k = case["rows"], case["classes"], case["k"]
        return {"bytes": n * (v * es + k * (es + 8) + 4), "flops": 3 * n * v}
    if case["kind"] in ("distill", "distill_one"):
        n, v, k = case["rows"], case["classes"], case["k"]
        entries = n * (k * (es + 8) + (4 if case["rest"] else 0))
        return {"bytes": 2 * n * v * es + entries + 4 * (n if case["reduction"] == "none" else 1), "flops": 7 * n * v}
    m, k, n = case["rows"], case["inputs"], case["outputs"]
    residual = m * n if case["residual"] != "none" else 0
    once = m * k + n * k + (n if case["bias"] else 0) + residual
    if case["kind"] == "linear":
        return {"bytes": es * (once + m * n), "flops": 2 * m * n * k}
    # every input read and its gradient written, the output written and its gradient read
    return {"bytes": es * (2 * once + 2 * m * n), "flops": 6 * m * n * k}


# ------------------------------------------------------------------ in 64 bits
def _exact_top(logits, k, t):
    """By one sortable key for each value and place: larger values first, then lower columns."""
    n, v = logits.shape
    bits = (logits.float() + 0.0).view(torch.int32).long()  # + 0.0: no negative zero
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    order = (key * v + (v - 1 - torch.arange(v, device=key.device))).topk(k, dim=1)[1]
    others = logits.double().div(t)
    others[torch.arange(n, device=order.device)[:, None], order] = -math.inf
    return {"values": logits.double().gather(1, order), "indices": order, "rest": others.logsumexp(1)}


def _exact_distill(state):
    case = state["case"]
    t, s = case["t"], state["logits"].detach().double().div(case["t"])
    n, v = s.shape
    rows = state["indices"][:, 0] >= 0  # a row's entries are all there, or none is
    at = state["indices"].clamp(min=0)
    teacher = state["values"].double().div(t)
    if state["rest"] is not None:
        teacher = torch.cat([teacher, state["rest"].double()[:, None]], 1)
    log_p = teacher.log_softmax(1)
    log_q = s.log_softmax(1)
    mine = log_q.gather(1, at)
    others = log_q.scatter(1, at, -math.inf)
    rest_q = others.logsumexp(1, keepdim=True)
    p = log_p.exp()
    student = torch.cat([mine, rest_q], 1)[:, :log_p.shape[1]]
    losses = (p * (log_p - student)).sum(1).mul(t * t) * rows
    if case["kind"] == "distill":
        weight = state["upstream"].double()
    else:
        weight = torch.tensor(state["scale"], dtype=torch.float64, device="cuda")
    loss = losses
    if case["reduction"] != "none":
        count = max(1, int(rows.sum())) if case["reduction"] == "mean" else 1
        loss, weight = losses.sum() / count, weight / count
    weight = (weight * rows * t)[:, None]
    p_rest = p[:, case["k"]:].sum(1, keepdim=True)
    # q_j (1 - p_rest / q_rest) off the list, q_j - p_j on it
    grad = others.exp() * (1 - p_rest / rest_q.exp())
    grad.scatter_(1, at, mine.exp() - p[:, :case["k"]])
    return {"loss": loss, "grad": grad * weight}


def _exact_linear(state):
    case = state["case"]
    get = {name: state[name].detach().double() for name in ("x", "weight", "bias", "residual") if state[name] is not None}
    z = torch.einsum("mk,nk->mn", get["x"], get["weight"]) + get.get("bias", 0.0)
    r = get.get("residual", 0.0)
    if case["residual"] == "before":
        z, r = z + r, 0.0
    if case["act"] == "relu":
        y, slope = z.relu(), (z > 0).double()
    elif case["act"] == "gelu":
        y = z * torch.special.ndtr(z)
        slope = torch.special.ndtr(z) + z * (-z.square() / 2).exp() / math.sqrt(2 * math.pi)
    elif case["act"] == "silu":
        y = z * z.sigmoid()
        slope = z.sigmoid() + z * z.sigmoid() * (-z).sigmoid()
    else:
        y, slope = z, 1.0
    y = y + r
    if case["kind"] == "linear":
        return {"y": y}
    gy = state["upstream"].double()
    gz = gy * slope
    out = {"y": y, "x": torch.einsum("mn,nk->mk", gz, get["weight"]), "weight": torch.einsum("mn,mk->nk", gz, get["x"])}
    if "bias" in get:
        out["bias"] = gz.sum(0)
    if "residual" in get:
        out["residual"] = gz if case["residual"] == "before" else gy
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "top":
        return _exact_top(state["logits"], case["k"], case["t"])
    if case["kind"] in ("distill", "distill_one"):
        return _exact_distill(state)
    return _exact_linear(state)
