"""Locate and load the native operator library.

Mirrors the reference loader (``muon_ascend950/_loader.py:1-50``):

* ``MUON_ASCEND950_LIBRARY`` names the operator library explicitly
  (``_loader.py:11-16``); otherwise the first ``_C*.so`` next to this package is
  used (``_loader.py:18-25``);
* ``torch.ops.load_library`` registers ``muon_ascend950::polar_step``
  (``_loader.py:39``), and a FakeTensor kernel is registered for tracing, tolerating
  an earlier registration (``_loader.py:41-48``);
* loading is idempotent (``_loader.py:7``, ``:30-31``, ``:49``).

Differences: the accelerator check asks for a ROCm build of torch instead of
``torch_npu``, and a missing library is a hard error (there is no CPU fallback).
"""

from __future__ import annotations

import os
from pathlib import Path

_LOADED = False


def _library_path() -> Path:
    configured = os.environ.get("MUON_ASCEND950_LIBRARY")
    if configured:
        path = Path(configured).expanduser().resolve()
        if not path.is_file():
            raise RuntimeError(f"MUON_ASCEND950_LIBRARY does not exist: {path}")
        return path

    package_dir = Path(__file__).resolve().parent
    candidates = sorted(package_dir.glob("_C*.so"))
    if not candidates:
        raise RuntimeError(
            "muon_ascend950 native library is missing. Build it in place with "
            "`python setup.py build_ext --inplace` for the current torch/ROCm environment."
        )
    return candidates[0]


def load_library() -> None:
    global _LOADED
    if _LOADED:
        return

    try:
        import torch
    except ImportError as exc:
        raise RuntimeError("muon_ascend950 requires torch built for ROCm") from exc
    if not getattr(torch.version, "hip", None):
        raise RuntimeError("muon_ascend950 requires torch built for ROCm (torch.version.hip is unset)")

    torch.ops.load_library(str(_library_path()))

    def fake_polar_step(x, a: float, b: float, c: float):
        return torch.empty_like(x, memory_format=torch.contiguous_format)

    def fake_polar_express(x, coefficients, normalize: bool):
        return torch.empty_like(x, memory_format=torch.contiguous_format)

    def fake_muon_update(param, grad, momentum_buffer, momentum, nesterov, coefficients, lr,
                         weight_decay, lr_scale):
        return None

    def fake_muon_update_list(params, grads, momentum_buffers, momentum, nesterov, coefficients,
                              lr, weight_decay, lr_scale):
        return None

    def fake_norms_forward(y, residual, post_weight, gate, scale, scale_value, pre_weight,
                           gate_kind, rows_per_sequence, post_norm, pre_norm, eps, save):
        rows = y.numel() // y.shape[-1]
        return (residual.new_empty(y.shape), y.new_empty(y.shape if pre_norm else (0,)),
                y.new_empty((rows if save else 0, 2), dtype=torch.float32))

    def fake_norms_backward(y, residual, post_weight, gate, scale, scale_value, pre_weight,
                            gate_kind, rows_per_sequence, post_norm, pre_norm, eps, stats,
                            d_residual_out, d_normed, wanted):
        def grad(t, bit):
            return y.new_empty((0,)) if t is None or not wanted & bit else t.new_empty(t.shape)

        return (y.new_empty(y.shape), residual.new_empty(y.shape), grad(post_weight, 1),
                grad(gate, 2), grad(scale, 4), grad(pre_weight, 8))

    def fake_distill_forward(logits, teacher_logits, teacher_indices, labels, temperature,
                             label_weight, save):
        rows = logits.numel() // logits.shape[-1]
        return (logits.new_empty(logits.shape[:-1], dtype=torch.float32),
                logits.new_empty((rows if save else 0, 4), dtype=torch.float32))

    def fake_distill_backward(logits, teacher_logits, teacher_indices, labels, temperature,
                              label_weight, stats, grad_loss):
        return logits.new_empty(logits.shape)

    def fake_distill_with_grad(logits, teacher_logits, teacher_indices, labels, temperature,
                               label_weight, grad_loss, grad_value, grad):
        return logits.new_empty(logits.shape[:-1], dtype=torch.float32)

    def held(like, rows, cols, block_rows):
        kb = -(-cols // 128)
        scales = (like.new_empty((kb, rows), dtype=torch.float32).t() if block_rows == 1 else
                  like.new_empty((-(-rows // 128), kb), dtype=torch.float32))
        return like.new_empty((rows, kb * 128), dtype=torch.float8_e4m3fn), scales

    def fake_quantize_fp8(x, block_rows):
        return held(x, x.shape[0], x.shape[1], block_rows)

    def fake_fp8_matmul(a, a_scales, b, b_scales, dtype):
        return a.new_empty((a.shape[0], b.shape[0]), dtype=dtype)

    def fake_fp8_linear(x, values, scales):
        return x.new_empty((*x.shape[:-1], values.shape[0]))

    def held_bytes(like, rows, cols, block_rows):
        width = -(-cols // 128) * 128
        scales = width // 128 * (rows if block_rows == 1 else -(-rows // 128))
        return like.new_empty((-(-rows * width // 256) * 256 + 4 * scales,), dtype=torch.uint8)

    def fake_fp8_linear_forward(x, weight, save):
        n, k = weight.shape
        xt = held_bytes(x, k, x.numel() // k, 1) if save & 1 else x.new_empty((0,))
        wt = held_bytes(x, k, n, 128) if save & 2 else x.new_empty((0,))
        return x.new_empty((*x.shape[:-1], n)), xt, wt

    def fake_fp8_linear_backward(dy, saved_x, saved_w, k, weight_dtype, wanted):
        dx = dy.new_empty((*dy.shape[:-1], k) if wanted & 1 else (0,))
        dw = dy.new_empty((dy.shape[-1], k) if wanted & 2 else (0,),
                          dtype=weight_dtype if wanted & 2 else dy.dtype)
        return dx, dw

    for name, fake in (("muon_ascend950::quantize_fp8", fake_quantize_fp8),
                       ("muon_ascend950::fp8_matmul", fake_fp8_matmul),
                       ("muon_ascend950::fp8_linear", fake_fp8_linear),
                       ("muon_ascend950::fp8_linear_forward", fake_fp8_linear_forward),
                       ("muon_ascend950::fp8_linear_backward", fake_fp8_linear_backward),
                       ("muon_ascend950::distill_forward", fake_distill_forward),
                       ("muon_ascend950::distill_backward", fake_distill_backward),
                       ("muon_ascend950::distill_with_grad", fake_distill_with_grad),
                       ("muon_ascend950::norms_forward", fake_norms_forward),
                       ("muon_ascend950::norms_backward", fake_norms_backward),
                       ("muon_ascend950::polar_step", fake_polar_step),
                       ("muon_ascend950::polar_step_tall", fake_polar_step),
                       ("muon_ascend950::polar_express", fake_polar_express),
                       ("muon_ascend950::muon_update", fake_muon_update),
                       ("muon_ascend950::muon_update_list", fake_muon_update_list)):
        try:
            torch.library.register_fake(name)(fake)
        except RuntimeError as exc:
            if "already has" not in str(exc):
                raise
    _LOADED = True
