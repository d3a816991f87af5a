"""Operators of a training step around the Muon update, on hand-written gfx950 kernels.

* ``block_norms`` — the norms before and after a block, with its gate and residual scale.

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

__all__ = ["block_norms"]

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
