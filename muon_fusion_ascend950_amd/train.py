"""Operators of a training step around the Muon update, on hand-written gfx950 kernels.

* ``block_norms`` — the norms before and after a block, with its gate and residual scale;
* ``distill_topk``, ``distill_topk_with_grad`` — the loss against a teacher's top logits,
  and loss and gradient in one pass;
* ``fp8_linear``, ``fp8_matmul``, ``quantize_fp8``, ``Fp8Blocks`` — products in 8-bit
  floating point (e4m3) with a scale for each block of 128.

``muon_update`` starts from the gradients of a model's matrices; these are pieces of the
forward and backward pass that produce them.  All take ROCm GPU tensors of float32 or
bfloat16, run on torch's current stream, compute in float32 and round each result once;
gradients come through autograd.  No reference counterpart: the reference leaves the
training step to its caller (README.md:130).
"""

from __future__ import annotations

import torch

from ._loader import load_library

load_library()

__all__ = ["Fp8Blocks", "block_norms", "distill_topk", "distill_topk_with_grad", "fp8_linear",
           "fp8_matmul", "quantize_fp8"]

_ops = torch.ops.muon_ascend950
_DTYPES = (torch.float32, torch.bfloat16)


def _check_tensor(name, t, device=None, dtypes=_DTYPES) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if device is None:
        if t.device.type != "cuda":
            raise ValueError(f"{name} must be on a ROCm GPU, got {t.device}")
    elif t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype not in dtypes:
        names = " or ".join(str(d) for d in dtypes)
        raise TypeError(f"{name} must use {names}, got {t.dtype}")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(
        isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------- norms
_GATE_NONE, _GATE_CHANNEL, _GATE_SEQUENCE, _GATE_TOKEN, _GATE_FULL = range(5)
_MAX_CHANNELS = 16384


def _gate_kind(shape, gate):
    """(kind, rows that share one gate vector) of a gate for y of `shape`."""
    got, d = tuple(gate.shape), shape[-1]
    if got and got[-1] == d and all(n == 1 for n in got[:-1]) and len(got) <= len(shape):
        # one vector for all rows; a single row's gate is the same thing
        return _GATE_CHANNEL, 1
    if got == shape:
        return _GATE_FULL, 1
    if got == shape[:-1] + (1,):
        return _GATE_TOKEN, 1
    if len(shape) >= 3 and got == shape[:1] + (1,) * (len(shape) - 2) + (d,):
        rows = 1
        for n in shape[1:-1]:
            rows *= n
        return _GATE_SEQUENCE, rows
    raise ValueError(f"gate of shape {got} does not fit y of shape {shape}: expected [D], "
                     "[..., 1], [B, 1, D] or y's own shape")


class _BlockNorms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, post_weight, gate, scale, pre_weight, options):
        value, kind, per_sequence, post_norm, pre_norm, eps = options
        out, normed, stats = _ops.norms_forward(y, residual, post_weight, gate, scale, value,
                                                pre_weight, kind, per_sequence, post_norm,
                                                pre_norm, eps, True)
        ctx.save_for_backward(y, residual, post_weight, gate, scale, pre_weight, stats)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return out, (normed if pre_norm else None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_normed):
        y, residual, post_weight, gate, scale, pre_weight, stats = ctx.saved_tensors
        value, kind, per_sequence, post_norm, pre_norm, eps = ctx.options
        need = ctx.needs_input_grad
        if d_out is None and d_normed is None:
            return (None,) * 7
        wanted = need[2] | need[3] << 1 | need[4] << 2 | need[5] << 3
        grads = _ops.norms_backward(y, residual, post_weight, gate, scale, value, pre_weight,
                                    kind, per_sequence, post_norm, pre_norm, eps, stats, d_out,
                                    d_normed, wanted)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None,)


def block_norms(y: torch.Tensor, residual: torch.Tensor, *, post_weight=None, gate=None,
                residual_scale=1.0, pre_weight=None, post_norm: bool = True,
                pre_norm: bool = True, eps: float = 1e-6):
    """Join a block's output to the residual stream and norm it for the next block::

        u = rms_norm(y, eps) * post_weight              # post_norm=False: u = y * post_weight
        residual_out = residual_scale * residual + gate * u
        normed = rms_norm(residual_out, eps) * pre_weight   # pre_norm=False: None

    Returns ``(residual_out, normed)``, of the dtypes of ``residual`` and ``y``.

    y, residual: one shape ``[..., D]``, D at most 16384; each float32 or bfloat16.
    post_weight, pre_weight: ``[D]`` of one dtype, or None (no weight).
    gate: None, ``[D]``, ``[..., 1]`` (per token), ``[B, 1, D]`` (per sequence of y
    ``[B, ..., D]``) or y's shape.  residual_scale: a number, or a float32 tensor of one
    or D elements.  Gradients of all tensors, those of broadcast ones summed.
    """
    _check_tensor("y", y)
    _check_tensor("residual", residual, y.device)
    if y.ndim < 1 or residual.shape != y.shape:
        raise ValueError(f"y and residual must have one shape [..., D], got {tuple(y.shape)} "
                         f"and {tuple(residual.shape)}")
    d = y.shape[-1]
    if not 1 <= d <= _MAX_CHANNELS:
        raise ValueError(f"D must be 1 to {_MAX_CHANNELS}, got {d}")
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is not None:
            _check_tensor(name, w, y.device)
            if w.shape != (d,):
                raise ValueError(f"{name} must have shape ({d},), got {tuple(w.shape)}")
    if post_weight is not None and pre_weight is not None and post_weight.dtype != pre_weight.dtype:
        raise TypeError("post_weight and pre_weight must have one dtype")
    if pre_weight is not None and not pre_norm:
        raise ValueError("pre_weight needs pre_norm")
    kind, per_sequence = _GATE_NONE, 1
    if gate is not None:
        _check_tensor("gate", gate, y.device)
        kind, per_sequence = _gate_kind(tuple(y.shape), gate)
    scale, value = None, 1.0
    if isinstance(residual_scale, torch.Tensor):
        _check_tensor("residual_scale", residual_scale, y.device, (torch.float32,))
        if tuple(residual_scale.shape) not in ((), (1,), (d,)):
            raise ValueError(f"residual_scale must have one or {d} elements, got shape "
                             f"{tuple(residual_scale.shape)}")
        scale = residual_scale
    else:
        value = float(residual_scale)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if _wants_grad(y, residual, post_weight, gate, scale, pre_weight):
        options = (value, kind, per_sequence, bool(post_norm), bool(pre_norm), float(eps))
        return _BlockNorms.apply(y, residual, post_weight, gate, scale, pre_weight, options)
    out, normed, _ = _ops.norms_forward(y, residual, post_weight, gate, scale, value, pre_weight,
                                        kind, per_sequence, bool(post_norm), bool(pre_norm),
                                        float(eps), False)
    return out, (normed if pre_norm else None)


# -------------------------------------------------------------------------- distillation
_MAX_TOP = 1024


class _DistillTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_indices, labels, temperature, label_weight):
        loss, stats = _ops.distill_forward(logits, teacher_logits, teacher_indices, labels,
                                           temperature, label_weight, True)
        ctx.save_for_backward(logits, teacher_logits, teacher_indices, labels, stats)
        ctx.options = temperature, label_weight
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, teacher_logits, teacher_indices, labels, stats = ctx.saved_tensors
        grad = _ops.distill_backward(logits, teacher_logits, teacher_indices, labels,
                                     *ctx.options, stats, grad_loss)
        return grad, None, None, None, None, None


def _check_distill(logits, teacher_logits, teacher_indices, temperature, labels, label_weight):
    """Checks the operands; returns (labels or None, temperature, label weight)."""
    _check_tensor("logits", logits)
    _check_tensor("teacher_logits", teacher_logits, logits.device)
    _check_tensor("teacher_indices", teacher_indices, logits.device, (torch.int32, torch.int64))
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape [..., V], got {tuple(logits.shape)}")
    if (teacher_logits.ndim != logits.ndim or teacher_logits.shape[:-1] != logits.shape[:-1]
            or teacher_indices.shape != teacher_logits.shape):
        raise ValueError(
            f"teacher_logits and teacher_indices must have shape {tuple(logits.shape[:-1])} + (K,), "
            f"got {tuple(teacher_logits.shape)} and {tuple(teacher_indices.shape)}")
    if not 1 <= teacher_logits.shape[-1] <= _MAX_TOP:
        raise ValueError(f"K must be 1 to {_MAX_TOP}, got {teacher_logits.shape[-1]}")
    temperature, label_weight = float(temperature), float(label_weight)
    if not 0.0 < temperature < 1e30:
        raise ValueError(f"temperature must be positive, got {temperature}")
    if not 0.0 <= label_weight <= 1.0:
        raise ValueError(f"label_weight must be 0 to 1, got {label_weight}")
    if labels is None:
        if label_weight != 0.0:
            raise ValueError("label_weight needs labels")
    else:
        _check_tensor("labels", labels, logits.device, (torch.int64,))
        if labels.shape != logits.shape[:-1]:
            raise ValueError(f"labels must have shape {tuple(logits.shape[:-1])}, "
                             f"got {tuple(labels.shape)}")
        if label_weight == 0.0:
            labels = None
    return labels, temperature, label_weight


def distill_topk(logits: torch.Tensor, teacher_logits: torch.Tensor,
                 teacher_indices: torch.Tensor, *, temperature: float = 1.0, labels=None,
                 label_weight: float = 0.0) -> torch.Tensor:
    """Loss of each row of student logits against a teacher's top logits::

        p = softmax(teacher_logits / temperature)       # over the row's K entries
        q = softmax(logits / temperature)               # over the vocabulary
        loss = (1 - label_weight) * temperature**2 * sum(p * (log p - log q[teacher_indices]))
               + label_weight * cross_entropy(logits, labels)

    logits ``[..., V]``, teacher_logits ``[..., K]`` (K at most 1024) float32 or bfloat16;
    teacher_indices ``[..., K]`` int32 or int64; labels ``[...]`` int64.  Returns float32
    ``[...]``, differentiable with respect to ``logits``.

    An entry whose index is outside ``[0, V)`` is absent (rows with fewer than K entries are
    filled with -1), and an absent entry's logit is not looked at.  A row without entries,
    or whose entries are all -inf, has no first term and no gradient from it; a label
    outside ``[0, V)`` (such as -100) leaves its row without the second.
    """
    labels, temperature, label_weight = _check_distill(
        logits, teacher_logits, teacher_indices, temperature, labels, label_weight)
    if _wants_grad(logits):
        return _DistillTopk.apply(logits, teacher_logits, teacher_indices, labels, temperature,
                                  label_weight)
    return _ops.distill_forward(logits, teacher_logits, teacher_indices, labels, temperature,
                                label_weight, False)[0]


@torch.no_grad()
def distill_topk_with_grad(logits: torch.Tensor, teacher_logits: torch.Tensor,
                           teacher_indices: torch.Tensor, *, grad_loss=1.0,
                           temperature: float = 1.0, labels=None, label_weight: float = 0.0,
                           out=None):
    """``distill_topk`` and its gradient in one pass over the logits.

    Returns ``(loss, grad)`` with ``grad`` the gradient of ``sum(grad_loss * loss)`` with
    respect to ``logits``, in their dtype, for ``logits.backward(grad)`` further down.
    grad_loss: a number or float32 ``[...]`` (0 for tokens that do not count).  ``out``
    receives the gradient; it may be ``logits`` itself, which is then overwritten.
    """
    labels, temperature, label_weight = _check_distill(
        logits, teacher_logits, teacher_indices, temperature, labels, label_weight)
    weight, value = None, 1.0
    if isinstance(grad_loss, torch.Tensor):
        _check_tensor("grad_loss", grad_loss, logits.device, (torch.float32,))
        if grad_loss.shape != logits.shape[:-1]:
            raise ValueError(f"grad_loss must have shape {tuple(logits.shape[:-1])}, "
                             f"got {tuple(grad_loss.shape)}")
        weight = grad_loss
    else:
        value = float(grad_loss)
    if out is None:
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
    else:
        _check_tensor("out", out, logits.device, (logits.dtype,))
        if out.shape != logits.shape:
            raise ValueError(f"out must have shape {tuple(logits.shape)}, got {tuple(out.shape)}")
        grad = out
    loss = _ops.distill_with_grad(logits, teacher_logits, teacher_indices, labels, temperature,
                                  label_weight, weight, value, grad)
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return loss, grad


# ---------------------------------------------------------------------------------- fp8
_BLOCK = 128


def _blocks(n: int) -> int:
    return -(-n // _BLOCK)


class Fp8Blocks:
    """A matrix as 8-bit values with a float32 scale for each block of 1 x 128 or 128 x 128.

    values: ``float8_e4m3fn [rows, cols rounded up to a multiple of 128]``, zero past
    ``cols`` (values of ``cols`` columns are padded here, by a copy); scales: float32
    ``[rows, ceil(cols / 128)]`` or ``[ceil(rows / 128), ceil(cols / 128)]``; shape:
    ``(rows, cols)``, by default that of ``values``.  Element (i, j) stands for
    ``values[i, j] * scales[i or i // 128, j // 128]``.
    """

    __slots__ = ("values", "scales", "shape")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, shape=None):
        _check_tensor("values", values, dtypes=(torch.float8_e4m3fn,))
        _check_tensor("scales", scales, values.device, (torch.float32,))
        if values.ndim != 2:
            raise ValueError(f"values must be a matrix, got shape {tuple(values.shape)}")
        rows, cols = tuple(values.shape) if shape is None else tuple(shape)
        if cols < 1:
            raise ValueError("a matrix must have columns")
        padded = _blocks(cols) * _BLOCK
        if rows != values.shape[0] or values.shape[1] not in (cols, padded):
            raise ValueError(f"values of shape {tuple(values.shape)} do not hold a matrix of shape "
                             f"{(rows, cols)}")
        if tuple(scales.shape) not in ((rows, _blocks(cols)), (_blocks(rows), _blocks(cols))):
            raise ValueError(f"scales must have shape {(rows, _blocks(cols))} or "
                             f"{(_blocks(rows), _blocks(cols))}, got {tuple(scales.shape)}")
        if values.shape[1] != padded:
            whole = torch.zeros(rows, padded, dtype=torch.uint8, device=values.device)
            whole[:, :cols] = values.view(torch.uint8)
            values = whole.view(torch.float8_e4m3fn)
        self.values, self.scales, self.shape = values, scales, (rows, cols)

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The matrix that the values and scales stand for."""
        rows, cols = self.shape
        scales = self.scales
        if scales.shape[0] != rows:
            scales = scales.repeat_interleave(_BLOCK, dim=0)[:rows]
        wide = scales.repeat_interleave(_BLOCK, dim=1)
        return (self.values.float() * wide)[:, :cols].to(dtype)


def quantize_fp8(x: torch.Tensor, block_rows: int = 1) -> Fp8Blocks:
    """``x`` ``[rows, cols]`` (float32 or bfloat16) in blocks of ``block_rows`` x 128, 1 for
    activations and gradients or 128 for weights::

        scale = max(amax(|block|) * (1 / 448), 2**-126)
        values = (block * (1 / scale)).to(float8_e4m3fn)

    A block that holds an infinity or a NaN has none but NaN back.
    """
    _check_tensor("x", x)
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError(f"x must have shape [rows, cols], got {tuple(x.shape)}")
    if block_rows not in (1, _BLOCK):
        raise ValueError(f"block_rows must be 1 or {_BLOCK}, got {block_rows}")
    values, scales = _ops.quantize_fp8(x.detach(), block_rows)
    return Fp8Blocks(values, scales, x.shape)


def _check_blocks(name, b) -> None:
    if not isinstance(b, Fp8Blocks):
        raise TypeError(f"{name} must be Fp8Blocks")


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T`` of matrices ``[M, K]`` and ``[N, K]``, summed in float32 and rounded once to
    ``dtype`` (float32 or bfloat16).  No gradient: see ``fp8_linear``."""
    _check_blocks("a", a)
    _check_blocks("b", b)
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"a and b must have one width, got {a.shape} and {b.shape}")
    if a.values.device != b.values.device:
        raise ValueError(f"b must be on {a.values.device}, got {b.values.device}")
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, got {dtype}")
    return _ops.fp8_matmul(a.values, a.scales, b.values, b.scales, dtype)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        need_x, need_w = ctx.needs_input_grad
        y, *saved = _ops.fp8_linear_forward(x, weight, need_w | need_x << 1)
        ctx.save_for_backward(*saved)
        ctx.weight_dtype = weight.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w = ctx.needs_input_grad
        dx, dw = _ops.fp8_linear_backward(dy, *ctx.saved_tensors, ctx.weight_dtype,
                                          need_x | need_w << 1)
        return dx if need_x else None, dw if need_w else None


def fp8_linear(x: torch.Tensor, weight) -> torch.Tensor:
    """``x @ weight.T`` in 8-bit floating point: x ``[..., K]`` quantised in blocks of 1 x 128,
    the weight ``[N, K]`` in blocks of 128 x 128; the result has x's dtype.

    weight: a float32 or bfloat16 matrix (training: quantised in this call, and with the
    gradients dx = dy @ weight and dweight = dy.T @ x, whose products are in 8 bits too, dy
    and x quantised in blocks of 128 along the axis that each product sums over), or
    ``Fp8Blocks`` (serving: no gradient).
    """
    _check_tensor("x", x)
    if x.ndim < 1:
        raise ValueError("x must have shape [..., K]")
    if isinstance(weight, Fp8Blocks):
        if weight.values.device != x.device:
            raise ValueError(f"weight must be on {x.device}, got {weight.values.device}")
        if weight.shape[1] != x.shape[-1]:
            raise ValueError(f"x must have {weight.shape[1]} columns, got shape {tuple(x.shape)}")
        if _wants_grad(x):
            raise ValueError("a quantised weight has no gradient: pass the float32 or bfloat16 one")
        return _ops.fp8_linear(x, weight.values, weight.scales)
    _check_tensor("weight", weight, x.device)
    if weight.ndim != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight must have shape [N, {x.shape[-1]}], got {tuple(weight.shape)}")
    if 0 in weight.shape:
        raise ValueError("weight's dimensions must be positive")
    if _wants_grad(x, weight):
        return _Fp8Linear.apply(x, weight)
    return _ops.fp8_linear_forward(x, weight, 0)[0]
