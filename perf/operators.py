"""Timed cases of the operators of a training step around the Muon update: the norms, gate
and residual scale around a block (``block_norms``), the loss against a teacher's top
logits (``distill_topk``) and products in 8-bit floating point with a scale for each block
of 128 (``fp8_linear``).

A case is a dict: ``op`` names the operator, the rest its sizes and options.  ``listed()``
are fixed cases, ``draw`` makes others over the same ranges.  With ``own`` false ``run``
computes the operators from elementary torch operations in 32 bits; with ``own`` true it
calls the package.  ``exact`` gives the results in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_DEV = "cuda"
_EPS = 1e-6
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_BLOCK = 128
_FP8_MAX = 448.0


def listed():
    return [
        # Decoding: one token's residual stream between two blocks.
        {"name": "norms_token", "op": "norms", "batch": 1, "seq": 1, "d": 4096, "dtype": "bfloat16",
         "residual": "bfloat16", "gate": "channel", "scale": "number", "train": False},
        # Prefill of a long prompt, residual stream kept in float32.
        {"name": "norms_prefill", "op": "norms", "batch": 1, "seq": 8192, "d": 4096,
         "dtype": "bfloat16", "residual": "float32", "gate": "none", "scale": "number",
         "train": False},
        # Training step, one gate vector for each sequence (conditioning), learned scale.
        {"name": "norms_train", "op": "norms", "batch": 4, "seq": 4096, "d": 4096,
         "dtype": "bfloat16", "residual": "bfloat16", "gate": "sequence", "scale": "scalar",
         "train": True},
        # A small model in float32 with odd sizes, a gate for each token, a scale vector.
        {"name": "norms_train_odd", "op": "norms", "batch": 7, "seq": 143, "d": 2051,
         "dtype": "float32", "residual": "float32", "gate": "token", "scale": "vector",
         "train": True},
        # Evaluation of a few tokens: rows are fewer than compute units.
        {"name": "distill_eval", "op": "distill", "rows": 8, "vocab": 32768, "k": 16,
         "dtype": "bfloat16", "tau": 1.0, "labels": False, "form": "loss"},
        # Training step, loss and gradient in one call; prompt tokens weigh nothing.
        {"name": "distill_train", "op": "distill", "rows": 8192, "vocab": 65536, "k": 64,
         "dtype": "bfloat16", "tau": 2.0, "labels": False, "form": "with_grad"},
        # Autograd's two calls on float32 logits of an odd, padded vocabulary, with labels.
        {"name": "distill_train_odd", "op": "distill", "rows": 1001, "vocab": 50001, "k": 20,
         "dtype": "float32", "tau": 1.5, "labels": True, "form": "autograd"},
        # Decoding: one token through an MLP up-projection, bound by the weight's bytes.
        {"name": "fp8_token", "op": "fp8", "tokens": 1, "n": 14336, "k": 4096,
         "dtype": "bfloat16", "train": False},
        # A short chunk of tokens through an odd projection.
        {"name": "fp8_chunk_odd", "op": "fp8", "tokens": 150, "n": 2050, "k": 1000,
         "dtype": "bfloat16", "train": False},
        # Prefill through an MLP up-projection (the largest case).
        {"name": "fp8_prefill", "op": "fp8", "tokens": 8192, "n": 14336, "k": 4096,
         "dtype": "bfloat16", "train": False},
        # Training step of an attention projection: forward and both gradients.
        {"name": "fp8_train", "op": "fp8", "tokens": 8192, "n": 4096, "k": 4096,
         "dtype": "bfloat16", "train": True},
        # The same at odd sizes, float32 activations.
        {"name": "fp8_train_odd", "op": "fp8", "tokens": 333, "n": 768, "k": 2050,
         "dtype": "float32", "train": True},
    ]


def draw(rng):
    def spread(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        # a third odd, a third in whole 64s, the rest as drawn
        kind = rng.randrange(3)
        return n | 1 if kind == 0 else max(1, n - n % 64) if kind == 1 and n > 64 else n

    while True:
        op = rng.choice(["norms", "distill", "fp8"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        if op == "norms":
            case = {"op": op, "batch": spread(1, 16), "seq": spread(1, 8192), "d": spread(64, 8192),
                    "dtype": dtype, "residual": rng.choice(["bfloat16", "float32"]),
                    "gate": rng.choice(["none", "channel", "sequence", "token", "full"]),
                    "scale": rng.choice(["number", "scalar", "vector"]),
                    "train": rng.random() < 0.6}
        elif op == "distill":
            case = {"op": op, "rows": spread(1, 8192), "vocab": spread(1000, 160000),
                    "k": min(spread(4, 256), 256), "dtype": dtype, "tau": rng.choice([1.0, 2.0, 1.5]),
                    "labels": rng.random() < 0.4,
                    "form": rng.choice(["loss", "with_grad", "autograd"])}
        else:
            case = {"op": op, "tokens": spread(1, 8192), "n": spread(128, 14336),
                    "k": spread(128, 14336), "dtype": dtype, "train": rng.random() < 0.5}
        w = work(case)
        if w["bytes"] <= 1.2e9 and w["flops"] <= 9e11:
            return case


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=_DEV, dtype=torch.float32).to(dtype)


def _gate_shape(case):
    b, s, d = case["batch"], case["seq"], case["d"]
    return {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, s, 1),
            "full": (b, s, d)}[case["gate"]]


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    if case["op"] == "norms":
        return _prepare_norms(case, gen)
    if case["op"] == "distill":
        return _prepare_distill(case, gen)
    return _prepare_fp8(case, gen)


def _prepare_norms(case, gen):
    b, s, d = case["batch"], case["seq"], case["d"]
    dtype, rdtype = _TYPES[case["dtype"]], _TYPES[case["residual"]]
    # a residual stream has a few channels far above the rest
    channel = torch.exp(0.5 * _randn(gen, d))
    channel[:: max(1, d // 4)] *= 20.0
    y = (_randn(gen, b, s, d) * 0.7).to(dtype)
    residual = (_randn(gen, b, s, d) * channel).to(rdtype)
    shape = _gate_shape(case)
    gate_type = torch.float32 if case["gate"] == "channel" else dtype
    state = {
        "op": "norms", "case": case, "y": y, "residual": residual,
        "post_weight": 1.0 + 0.2 * _randn(gen, d), "pre_weight": 1.0 + 0.2 * _randn(gen, d),
        "gate": None if shape is None else (0.5 + 0.5 * _randn(gen, *shape)).to(gate_type),
        "scale": {"number": 0.9, "scalar": 0.9 + 0.05 * _randn(gen, 1),
                  "vector": 0.9 + 0.05 * _randn(gen, d)}[case["scale"]],
    }
    if case["train"]:
        state["d_residual"] = (_randn(gen, b, s, d) * 1e-3).to(rdtype)
        state["d_normed"] = (_randn(gen, b, s, d) * 1e-3).to(dtype)
        for name in _learned(state):
            state[name].requires_grad_(True)
    return state


def _learned(state):
    """The tensors that a training step takes gradients of, in the order of its outputs."""
    names = ["y", "residual", "post_weight", "pre_weight"]
    return names + [n for n in ("gate", "scale") if isinstance(state[n], torch.Tensor)]


def _prepare_distill(case, gen):
    t, v, k = case["rows"], case["vocab"], case["k"]
    dtype = _TYPES[case["dtype"]]
    base = _randn(gen, t, v, dtype=torch.bfloat16)
    logits = (2.0 * base).to(dtype)
    # the teacher agrees with the student in part
    teacher = base.mul_(1.5).add_(_randn(gen, t, v, dtype=torch.bfloat16))
    odd = v % 2 == 1
    if odd:  # a vocabulary padded for its layout: the padding is masked
        logits[:, -5:] = -math.inf
        teacher[:, -5:] = -math.inf
    top, index = torch.topk(teacher, k, dim=1)
    if odd:  # stored top entries of unequal count: -1 where a row has fewer
        count = torch.randint(1, k + 1, (t, 1), generator=gen, device=_DEV)
        index = torch.where(torch.arange(k, device=_DEV) < count, index, -1)
    weight = (torch.rand(t, generator=gen, device=_DEV) > 0.25).float() / max(1, t)
    state = {"op": "distill", "case": case, "logits": logits, "teacher": top,
             "index": index.to(torch.int32), "weight": weight, "labels": None, "lam": 0.0}
    if case["labels"]:
        labels = torch.randint(0, v - 5, (t,), generator=gen, device=_DEV)
        state["labels"] = torch.where(torch.rand(t, generator=gen, device=_DEV) < 0.1, -100, labels)
        state["lam"] = 0.25
    if case["form"] == "autograd":
        logits.requires_grad_(True)
    return state


def _quantize(x, rows):
    """x [R, C] in blocks of `rows` x 128: values as float8 [R, C padded to 128s], zero
    there, and float32 scales [ceil(R / rows), ceil(C / 128)]."""
    r, c = x.shape
    rp, cp = -(-r // rows) * rows, -(-c // _BLOCK) * _BLOCK
    xp = torch.nn.functional.pad(x.float(), (0, cp - c, 0, rp - r))
    blocks = xp.view(rp // rows, rows, cp // _BLOCK, _BLOCK)
    scales = (blocks.abs().amax(dim=(1, 3)) * (1.0 / _FP8_MAX)).clamp_min(2.0 ** -126)
    values = (blocks * torch.reciprocal(scales)[:, None, :, None]).to(torch.float8_e4m3fn)
    return values.view(rp, cp)[:r], scales


def _dequantize(values, scales, rows, dtype=torch.float32):
    r, c = values.shape
    s = scales.to(dtype).repeat_interleave(rows, dim=0)[:r].repeat_interleave(_BLOCK, dim=1)
    return values.to(dtype) * s


def _prepare_fp8(case, gen):
    t, n, k = case["tokens"], case["n"], case["k"]
    dtype = _TYPES[case["dtype"]]
    channel = torch.exp(0.5 * _randn(gen, k))
    channel[:: max(1, k // 8)] *= 15.0  # outlying channels of the activations
    x = (_randn(gen, t, k) * channel).to(dtype)
    weight = _randn(gen, n, k) / math.sqrt(k)
    state = {"op": "fp8", "case": case, "x": x}
    if case["train"]:
        state["weight"] = weight.requires_grad_(True)
        # gradients of tokens differ in size by orders of magnitude
        state["d_y"] = (_randn(gen, t, n) * 1e-4 * torch.exp(_randn(gen, t, 1))).to(dtype)
        x.requires_grad_(True)
    else:  # a server keeps the quantised weight
        state["values"], state["scales"] = _quantize(weight, _BLOCK)
    return state


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norms": _plain_norms, "distill": _plain_distill, "fp8": _plain_fp8}[state["op"]](state)


def _run_own(state):
    from muon_fusion_ascend950_amd import train

    case = state["case"]
    if state["op"] == "norms":
        out = train.block_norms(state["y"], state["residual"], post_weight=state["post_weight"],
                                gate=state["gate"], residual_scale=state["scale"],
                                pre_weight=state["pre_weight"], eps=_EPS)
        if not case["train"]:
            return out
        grads = torch.autograd.grad(out, [state[n] for n in _learned(state)],
                                    [state["d_residual"], state["d_normed"]])
        return tuple(t.detach() for t in out) + grads
    if state["op"] == "distill":
        args = (state["logits"], state["teacher"], state["index"])
        options = {"temperature": case["tau"], "labels": state["labels"],
                   "label_weight": state["lam"]}
        if case["form"] == "loss":
            return train.distill_topk(*args, **options)
        if case["form"] == "with_grad":
            return train.distill_topk_with_grad(*args, grad_loss=state["weight"], **options)
        loss = train.distill_topk(*args, **options)
        (grad,) = torch.autograd.grad(loss, state["logits"], state["weight"])
        return loss.detach(), grad
    if not case["train"]:
        weight = train.Fp8Blocks(state["values"], state["scales"], (case["n"], case["k"]))
        return train.fp8_linear(state["x"], weight)
    y = train.fp8_linear(state["x"], state["weight"])
    grads = torch.autograd.grad(y, (state["x"], state["weight"]), state["d_y"])
    return (y.detach(),) + grads


# ------------------------------------------------------------------ plain forms, 32 bits
def _sum_to(t, like):
    """t summed over the axes along which `like` was broadcast, in like's shape and type."""
    shape = (1,) * (t.dim() - like.dim()) + tuple(like.shape)
    axes = [i for i, n in enumerate(shape) if n == 1 and t.shape[i] != 1]
    return (t.sum(dim=axes, keepdim=True) if axes else t).reshape(like.shape).to(like.dtype)


def _plain_norms(state):
    y, r = state["y"].float(), state["residual"].float()
    w1, w2 = state["post_weight"], state["pre_weight"]
    gate, scale = state["gate"], state["scale"]
    alpha = scale
    g = 1.0 if gate is None else gate.float()
    rho1 = torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + _EPS)
    n = y * rho1
    u = n * w1
    total = alpha * r + g * u
    rho2 = torch.rsqrt((total * total).mean(dim=-1, keepdim=True) + _EPS)
    m = total * rho2
    out = (total.to(state["residual"].dtype), (m * w2).to(state["y"].dtype))
    if not state["case"]["train"]:
        return out
    dh = state["d_normed"].float()
    dm = dh * w2
    dt = state["d_residual"].float() + rho2 * (dm - m * (dm * m).mean(dim=-1, keepdim=True))
    du = dt * g
    dn = du * w1
    dy = rho1 * (dn - n * (dn * n).mean(dim=-1, keepdim=True))
    grads = (dy.to(state["y"].dtype), (alpha * dt).to(state["residual"].dtype),
             _sum_to(du * n, w1), _sum_to(dh * m, w2))
    if gate is not None:
        grads += (_sum_to(dt * u, gate),)
    if isinstance(scale, torch.Tensor):
        grads += (_sum_to(dt * r, scale),)
    return out + grads


def _plain_distill(state):
    case, tau, lam = state["case"], state["case"]["tau"], state["lam"]
    logits, index, labels = state["logits"], state["index"].long(), state["labels"]
    present = index >= 0
    safe = index.clamp_min(0)
    z = logits.float() / tau
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    log_q = z.gather(1, safe) - top - torch.log(total)
    t = torch.where(present, state["teacher"].float() / tau, -math.inf)
    pe = torch.exp(t - t.amax(dim=1, keepdim=True))
    pe = torch.where(present, pe, 0.0)
    psum = pe.sum(dim=1, keepdim=True)
    p = pe / psum
    log_p = t - t.amax(dim=1, keepdim=True) - torch.log(psum)
    loss = (1.0 - lam) * tau * tau * torch.where(p > 0, p * (log_p - log_q), 0.0).sum(dim=1)
    if labels is not None:
        z1 = logits.float()
        top1 = z1.amax(dim=1, keepdim=True)
        e1 = torch.exp(z1 - top1)
        total1 = e1.sum(dim=1, keepdim=True)
        known = labels != -100
        at = labels.clamp_min(0)[:, None]
        ce = (top1 + torch.log(total1) - z1.gather(1, at))[:, 0]
        loss = loss + lam * torch.where(known, ce, 0.0)
    if case["form"] == "loss":
        return loss
    w = state["weight"][:, None]
    grad = e.div_(total)
    grad.scatter_add_(1, safe, -p)
    grad.mul_((1.0 - lam) * tau)
    if labels is not None:
        hard = e1.div_(total1)
        hard.scatter_add_(1, at, torch.full_like(w, -1.0))
        grad.add_(torch.where(known[:, None], hard, 0.0), alpha=lam)
    return loss, grad.mul_(w).to(logits.dtype)


def _plain_fp8(state):
    x = state["x"]
    xd = _dequantize(*_quantize(x, 1), 1)
    if not state["case"]["train"]:
        return (xd @ _dequantize(state["values"], state["scales"], _BLOCK).t()).to(x.dtype)
    t, (n, k) = x.shape[0], state["weight"].shape
    wd = _dequantize(*_quantize(state["weight"], _BLOCK), _BLOCK)
    dy = state["d_y"]
    y = (xd @ wd.t()).to(x.dtype)
    dx = _dequantize(*_quantize(dy, 1), 1)[:, :n] @ wd[:, :k]
    along = _dequantize(*_quantize(dy.t(), 1), 1)  # quantised along the tokens
    dw = along @ _dequantize(*_quantize(x.t(), 1), 1).t()
    return y, dx.to(x.dtype), dw


# ------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"norms": _exact_norms, "distill": _exact_distill, "fp8": _exact_fp8}[case["op"]](state)


def _leaf(t):
    return t.detach().double().requires_grad_(True)


def _exact_norms(state):
    v = {n: _leaf(state[n]) for n in _learned(state)}
    v = {**{n: state[n] for n in ("gate", "scale")}, **v}

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * w

    with torch.enable_grad():
        branch = norm(v["y"], v["post_weight"])
        if v["gate"] is not None:
            branch = branch * v["gate"]
        total = v["residual"] * v["scale"] + branch
        out = (total, norm(total, v["pre_weight"]))
        if not state["case"]["train"]:
            return tuple(o.detach() for o in out)
        grads = torch.autograd.grad(out, [v[n] for n in _learned(state)],
                                    [state["d_residual"].double(), state["d_normed"].double()])
    return tuple(o.detach() for o in out) + grads


def _exact_distill(state):
    tau, lam = state["case"]["tau"], state["lam"]
    z = _leaf(state["logits"])
    present = state["index"] >= 0
    at = torch.where(present, state["index"], 0).long()
    with torch.enable_grad():
        p = torch.softmax((state["teacher"].double() / tau).masked_fill(~present, -math.inf), dim=1)
        log_q = torch.log_softmax(z / tau, dim=1).gather(1, at)
        # p·(log p − log q); absent entries have p = 0
        terms = torch.special.xlogy(p, p) - p * log_q.masked_fill(~present, 0.0)
        loss = (1.0 - lam) * tau * tau * terms.sum(dim=1)
        if state["labels"] is not None:
            loss = loss + lam * torch.nn.functional.cross_entropy(
                z, state["labels"], ignore_index=-100, reduction="none")
        if state["case"]["form"] == "loss":
            return loss.detach()
        (grad,) = torch.autograd.grad(loss, z, state["weight"].double())
    return loss.detach(), grad


def _exact_fp8(state):
    # the 8-bit values and their scales are the operator's own definition, in float32
    def held(x, rows):
        return _dequantize(*_quantize(x.detach(), rows), rows, torch.float64)

    x = held(state["x"], 1)
    if not state["case"]["train"]:
        return x @ _dequantize(state["values"], state["scales"], _BLOCK, torch.float64).t()
    n, k = state["weight"].shape
    w, dy = held(state["weight"], _BLOCK), state["d_y"]
    return (x @ w.t(), (held(dy, 1)[:, :n] @ w)[:, :k],
            held(dy.t().contiguous(), 1) @ held(state["x"].t().contiguous(), 1).t())


# ---------------------------------------------------------------------------------- work
def work(case):
    """Bytes (each input read once, each output written once) and operations of one pass."""
    size = {"float32": 4, "bfloat16": 2}
    if case["op"] == "norms":
        rows, d = case["batch"] * case["seq"], case["d"]
        sy, sr = size[case["dtype"]], size[case["residual"]]
        shape = _gate_shape(case)
        gate = 0 if shape is None else math.prod(shape) * (4 if case["gate"] == "channel" else sy)
        scale = {"number": 0, "scalar": 4, "vector": 4 * d}[case["scale"]]
        forward = 2 * rows * d * (sy + sr) + 8 * d + gate + scale
        if not case["train"]:
            return {"bytes": forward, "flops": 12 * rows * d}
        # the backward pass reads the inputs and the two gradients and writes its own
        backward = 3 * rows * d * (sy + sr) + 2 * (8 * d + gate + scale)
        return {"bytes": forward + backward, "flops": 40 * rows * d}
    if case["op"] == "distill":
        t, v, k = case["rows"], case["vocab"], case["k"]
        table = t * v * size[case["dtype"]]
        passes = {"loss": 1, "with_grad": 2, "autograd": 3}[case["form"]]
        top = t * k * 6 + 4 * t * (3 if case["labels"] else 2)
        return {"bytes": passes * table + top, "flops": 5 * passes * t * v}
    t, n, k = case["tokens"], case["n"], case["k"]
    s = size[case["dtype"]]
    if not case["train"]:
        return {"bytes": t * k * s + n * k + 4 * math.ceil(n / _BLOCK) * math.ceil(k / _BLOCK)
                + t * n * s, "flops": 2 * t * n * k}
    # x, weight, dy read once; y, dx, dw written once
    return {"bytes": 2 * t * (n + k) * s + 8 * n * k, "flops": 6 * t * n * k}
