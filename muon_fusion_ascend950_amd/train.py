"""Operators of a training step around the Muon update, on hand-written gfx950 kernels.

* ``block_norms`` — the norms before and after a block, with its gate and residual scale;
* ``distill_topk``, ``distill_topk_with_grad`` — the loss against a teacher's top logits,
  and loss and gradient in one pass;
* ``fp8_linear``, ``fp8_matmul``, ``quantize_fp8``, ``Fp8Blocks`` — products in 8-bit
  floating point (e4m3) with a scale for each block of 128.

``muon_update`` starts from the gradients of a model's matrices; these are pieces of the
forward and backward pass that produce them.  All take ROCm GPU tensors of float32 or
bfloat16, run on torch's current stream, compute in float32 (8-bit products with bfloat16
results: see ``fp8_matmul``) and round each result once;
gradients come through autograd, in reverse mode once (a gradient of a gradient and
forward-mode tangents are refused).  No reference counterpart: the reference leaves the
training step to its caller (README.md:130).
"""

from __future__ import annotations

import torch

from ._loader import load_library

load_library()

__all__ = ["Fp8Blocks", "block_norms", "distill_topk", "distill_topk_with_grad", "fp8_linear",
           "fp8_matmul", "quantize_fp8"]

_ops = torch.ops.muon_ascend950
_block_norms = _ops.block_norms.default
_distill_topk = _ops.distill_topk.default
_distill_topk_with_grad = _ops.distill_topk_with_grad.default
_fp8_linear_train = _ops.fp8_linear_train.default
_fp8_linear_serve = _ops.fp8_linear_serve.default
_DTYPES = (torch.float32, torch.bfloat16)


def _blame(required, optional) -> None:
    """After an operator refused its arguments: the one that is no tensor, if any (the
    operators check the rest; looking first would cost every call a microsecond)."""
    for name, t in {**required, **optional}.items():
        if not isinstance(t, torch.Tensor) and (t is not None or name in required):
            raise TypeError(f"{name} must be a torch.Tensor") from None


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
    scale, value = None, 1.0
    if isinstance(residual_scale, torch.Tensor):
        scale = residual_scale
    else:
        value = float(residual_scale)
    try:
        out, normed = _block_norms(y, residual, post_weight, gate, scale, value, pre_weight,
                                   post_norm, pre_norm, eps)
    except Exception:
        _blame(dict(y=y, residual=residual),
               dict(post_weight=post_weight, gate=gate, pre_weight=pre_weight))
        raise
    return out, (normed if pre_norm else None)


# -------------------------------------------------------------------------- distillation
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
    ``[...]``, differentiable with respect to ``logits``.  temperature: at least float32's
    smallest normal number, below 1e30.

    An entry whose index is outside ``[0, V)`` is absent (rows with fewer than K entries are
    filled with -1), and an absent entry's logit is not looked at.  A row without entries,
    or whose entries are all -inf, has no first term and no gradient from it; a label
    outside ``[0, V)`` (such as -100) leaves its row without the second.
    """
    try:
        return _distill_topk(logits, teacher_logits, teacher_indices, labels, temperature,
                             label_weight)
    except Exception:
        _blame(dict(logits=logits, teacher_logits=teacher_logits, teacher_indices=teacher_indices),
               dict(labels=labels))
        raise


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
    weight, value = None, 1.0
    if isinstance(grad_loss, torch.Tensor):
        weight = grad_loss
    else:
        value = float(grad_loss)
    try:
        loss, grad = _distill_topk_with_grad(logits, teacher_logits, teacher_indices, labels,
                                             temperature, label_weight, weight, value, out)
    except Exception:
        _blame(dict(logits=logits, teacher_logits=teacher_logits, teacher_indices=teacher_indices),
               dict(labels=labels, out=out))
        raise
    return loss, (grad if out is None else out)


# ---------------------------------------------------------------------------------- fp8
_BLOCK = 128


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

    A block that holds an infinity or a NaN has none but NaN back.  No gradient: ``x`` is
    taken detached.
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
    """``a @ b.T`` of matrices ``[M, K]`` and ``[N, K]``, rounded once to ``dtype`` (float32 or
    bfloat16).  No gradient: see ``fp8_linear``.

    float32 results are sums in float32.  For bfloat16 ones the matrix unit adds eight products
    of values at a time, each cut off below 2**-13 of the largest of them (off by 1.5e-5 to
    7e-5 of a result's norm as measured, at most 7 * 2**-13 of the sum of magnitudes); the sums
    of blocks of 128 are added in float32.
    """
    _check_blocks("a", a)
    _check_blocks("b", b)
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"a and b must have one width, got {a.shape} and {b.shape}")
    if a.values.device != b.values.device:
        raise ValueError(f"b must be on {a.values.device}, got {b.values.device}")
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, got {dtype}")
    return _ops.fp8_matmul(a.values, a.scales, b.values, b.scales, dtype)


def fp8_linear(x: torch.Tensor, weight) -> torch.Tensor:
    """``x @ weight.T`` in 8-bit floating point: x ``[..., K]`` quantised in blocks of 1 x 128,
    the weight ``[N, K]`` in blocks of 128 x 128; the result has x's dtype.  Sums are those of
    ``fp8_matmul`` for the dtype of each result (x's, and the weight's for its gradient).

    weight: a float32 or bfloat16 matrix (training: quantised in this call, and with the
    gradients dx = dy @ weight and dweight = dy.T @ x, whose products are in 8 bits too, dy
    and x quantised in blocks of 128 along the axis that each product sums over), or
    ``Fp8Blocks`` (serving: no gradient).  A call whose weight wants a gradient takes up to 2**22
    tokens, and tokens * max(N, K) up to about 2**35; one whose x does, tokens * N.
    """
    try:
        if isinstance(weight, Fp8Blocks):
            return _fp8_linear_serve(x, weight.values, weight.scales, weight.shape[1])
        return _fp8_linear_train(x, weight)
    except Exception:
        _blame(dict(x=x), {})
        if not isinstance(weight, (torch.Tensor, Fp8Blocks)):
            raise TypeError("weight must be a torch.Tensor or Fp8Blocks") from None
        raise
