"""Host side of the training-step operators, without a GPU: public names, refusals of wrong
arguments, FakeTensor kernels, and the C ABI of include/muon_train.h (its exported set and
its checks before any launch)."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import muon_fusion_ascend950_amd as mf
from muon_fusion_ascend950_amd import capi, train

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "muon_train.h"
F32, B16 = torch.float32, torch.bfloat16


def test_public_names():
    assert mf.train is train
    for name in train.__all__:
        assert getattr(train, name).__doc__, name


def test_header_declares_what_the_library_exports():
    declared = set(re.findall(r"^int (muon_train_\w+)\s*\(", HEADER.read_text(), re.M))
    out = subprocess.run(["nm", "-D", "--defined-only", str(capi.library_path())],
                         capture_output=True, text=True, check=True).stdout
    assert declared and declared == set(re.findall(r" T (muon_train_\w+)$", out, re.M))


# ------------------------------------------------------------------------------- norms
def _cuda(*shape, dtype=F32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _norms_ok(**change):
    args = dict(y=_cuda(2, 3, 64, dtype=B16), residual=_cuda(2, 3, 64), post_weight=_cuda(64),
                gate=_cuda(2, 1, 64, dtype=B16), residual_scale=_cuda(1), pre_weight=_cuda(64))
    args.update(change)
    return args


def _norms(**args):
    return train.block_norms(args.pop("y"), args.pop("residual"), **args)


@pytest.mark.parametrize("change,error,message", [
    (lambda: dict(y=[1.0]), TypeError, "torch.Tensor"),
    (lambda: dict(y=torch.zeros(2, 3, 64)), ValueError, "ROCm GPU"),
    (lambda: dict(y=_cuda(2, 3, 64, dtype=torch.float16)), TypeError, "float32 or torch.bfloat16"),
    (lambda: dict(residual=_cuda(2, 64)), ValueError, "one shape"),
    (lambda: dict(residual=torch.zeros(2, 3, 64)), ValueError, "cuda"),
    (lambda: dict(y=_cuda(2, 16385), residual=_cuda(2, 16385)), ValueError, "16384"),
    (lambda: dict(y=_cuda(2, 0), residual=_cuda(2, 0)), ValueError, "16384"),
    (lambda: dict(y=_cuda(), residual=_cuda()), ValueError, "shape"),
    (lambda: dict(post_weight=_cuda(63)), ValueError, "post_weight"),
    (lambda: dict(pre_weight=_cuda(1, 64)), ValueError, "pre_weight"),
    (lambda: dict(pre_weight=_cuda(64, dtype=B16)), TypeError, "one dtype"),
    (lambda: dict(pre_norm=False), ValueError, "pre_norm"),
    (lambda: dict(gate=_cuda(3, 1, 64)), ValueError, "gate"),
    (lambda: dict(gate=_cuda(2, 3)), ValueError, "gate"),
    (lambda: dict(gate=0.5), TypeError, "gate"),
    (lambda: dict(residual_scale=_cuda(2)), ValueError, "residual_scale"),
    (lambda: dict(residual_scale=_cuda(64, dtype=B16)), TypeError, "residual_scale"),
    (lambda: dict(eps=-1.0), ValueError, "eps"),
    (lambda: dict(eps=float("nan")), ValueError, "eps"),
])
def test_block_norms_refuses(change, error, message):
    with FakeTensorMode():
        with pytest.raises(error, match=message):
            _norms(**_norms_ok(**change()))


def test_block_norms_fake():
    with FakeTensorMode():
        args = _norms_ok()
        out, h = _norms(**args)
        assert out.shape == h.shape == (2, 3, 64) and (out.dtype, h.dtype) == (F32, B16)
        args = _norms_ok(pre_weight=None, pre_norm=False)
        assert _norms(**args)[1] is None
        args = _norms_ok()
        ops = torch.ops.muon_ascend950
        common = (args["y"], args["residual"], args["post_weight"], args["gate"],
                  args["residual_scale"], 1.0, args["pre_weight"], 2, 3, True, True, 1e-6)
        stats = ops.norms_forward(*common, True)[2]
        assert stats.shape == (6, 2) and stats.dtype == F32
        grads = ops.norms_backward(*common, stats, None, args["y"], 2 | 4)
        like = [args[n] for n in ("y", "residual", "gate", "residual_scale")]
        got = [grads[0], grads[1], grads[3], grads[4]]
        assert [(g.shape, g.dtype) for g in got] == [(t.shape, t.dtype) for t in like]
        assert grads[2].numel() == grads[5].numel() == 0


class NormsArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("rows", "d", "rows_per_sequence", "ld_y", "ld_residual")] + [
        (n, ctypes.c_void_p) for n in ("y", "residual", "post_weight", "pre_weight", "gate", "scale")] + [
        (n, ctypes.c_double) for n in ("scale_value", "eps")] + [
        (n, ctypes.c_int) for n in ("y_dtype", "residual_dtype", "weight_dtype", "gate_dtype",
                                    "gate_kind", "scale_kind", "post_norm", "pre_norm")] + [
        (n, ctypes.c_void_p) for n in ("residual_out", "normed", "stats", "d_residual_out", "d_normed",
                                       "d_y", "d_residual", "d_post_weight", "d_pre_weight",
                                       "d_gate", "d_scale")]


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows"), (dict(d=0), "d must"), (dict(d=16385), "d must"),
    (dict(y_dtype=2), "dtypes"), (dict(gate_kind=5), "kind"), (dict(scale_kind=-1), "kind"),
    (dict(gate_kind=2, rows_per_sequence=0, gate=4096), "rows_per_sequence"),
    (dict(gate_kind=2, rows_per_sequence=3, gate=4096), "rows_per_sequence"),
    (dict(gate_kind=1), "null"), (dict(scale_kind=1), "null"), (dict(y=None), "null"),
    (dict(ld_y=7), "overlap"), (dict(residual_out=None), "null output"),
    (dict(normed=None), "null output"), (dict(normed=(1 << 20) + 124), "overlap"),
    (dict(residual_out=(1 << 21) - 124), "overlap"), (dict(normed=(1 << 22) + 64), "overlap"),
])
def test_norms_entry_checks_before_any_launch(change, message):
    lib = capi.load()
    base = dict(rows=4, d=8, rows_per_sequence=4, ld_y=8, ld_residual=8, y=1 << 20, residual=1 << 21,
                eps=1e-6, pre_norm=1, residual_out=1 << 22, normed=1 << 23)
    args = NormsArgs(**{**base, **change})
    assert lib.muon_train_norms_forward(ctypes.byref(args), None) == capi.ERR_INVALID_ARGUMENT
    assert message in capi.last_error()
    assert lib.muon_train_norms_forward(None, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.muon_train_norms_forward(ctypes.byref(NormsArgs(**{**base, "rows": 0})), None) == capi.OK


# ------------------------------------------------------------------------ distillation
def _distill_ok(**change):
    args = dict(logits=_cuda(2, 3, 50, dtype=B16), teacher_logits=_cuda(2, 3, 4),
                teacher_indices=_cuda(2, 3, 4, dtype=torch.int32), temperature=2.0,
                labels=_cuda(2, 3, dtype=torch.int64), label_weight=0.5)
    args.update(change)
    return [args.pop(n) for n in ("logits", "teacher_logits", "teacher_indices")], args


@pytest.mark.parametrize("change,error,message", [
    (lambda: dict(logits=1.0), TypeError, "torch.Tensor"),
    (lambda: dict(logits=torch.zeros(2, 3, 50)), ValueError, "ROCm GPU"),
    (lambda: dict(logits=_cuda(2, 3, 50, dtype=torch.float16)), TypeError, "logits"),
    (lambda: dict(logits=_cuda(2, 3, 0)), ValueError, "logits"),
    (lambda: dict(logits=_cuda(6, 50)), ValueError, "teacher_logits"),
    (lambda: dict(logits=_cuda(2, 4, 50)), ValueError, "teacher_logits"),
    (lambda: dict(teacher_indices=_cuda(2, 3, 5, dtype=torch.int32)), ValueError, "teacher_indices"),
    (lambda: dict(teacher_indices=_cuda(2, 3, 4)), TypeError, "teacher_indices"),
    (lambda: dict(teacher_logits=_cuda(2, 3, 1025), teacher_indices=_cuda(2, 3, 1025, dtype=torch.int32)),
     ValueError, "1024"),
    (lambda: dict(teacher_logits=_cuda(2, 3, 0), teacher_indices=_cuda(2, 3, 0, dtype=torch.int32)),
     ValueError, "1024"),
    (lambda: dict(temperature=0.0), ValueError, "temperature"),
    (lambda: dict(temperature=float("nan")), ValueError, "temperature"),
    (lambda: dict(temperature=float("inf")), ValueError, "temperature"),
    (lambda: dict(label_weight=1.5), ValueError, "label_weight"),
    (lambda: dict(labels=None), ValueError, "labels"),
    (lambda: dict(labels=_cuda(2, dtype=torch.int64)), ValueError, "labels"),
    (lambda: dict(labels=_cuda(2, 3, dtype=torch.int32)), TypeError, "labels"),
])
def test_distill_refuses(change, error, message):
    with FakeTensorMode():
        for call in (train.distill_topk, train.distill_topk_with_grad):
            args, kw = _distill_ok(**change())
            with pytest.raises(error, match=message):
                call(*args, **kw)


def test_distill_with_grad_refuses_and_fake():
    with FakeTensorMode():
        args, kw = _distill_ok()
        with pytest.raises(ValueError, match="grad_loss"):
            train.distill_topk_with_grad(*args, grad_loss=_cuda(6), **kw)
        with pytest.raises(TypeError, match="grad_loss"):
            train.distill_topk_with_grad(*args, grad_loss=_cuda(2, 3, dtype=B16), **kw)
        with pytest.raises(TypeError, match="out"):
            train.distill_topk_with_grad(*args, out=_cuda(2, 3, 50), **kw)
        with pytest.raises(ValueError, match="out"):
            train.distill_topk_with_grad(*args, out=_cuda(6, 50, dtype=B16), **kw)
        loss, grad = train.distill_topk_with_grad(*args, **kw)
        assert (loss.shape, loss.dtype) == ((2, 3), F32)
        assert (grad.shape, grad.dtype) == ((2, 3, 50), B16)
        args[0].requires_grad_(True)
        loss = train.distill_topk(*args, **kw)
        assert (loss.shape, loss.dtype, loss.requires_grad) == ((2, 3), F32, True)


class DistillArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("rows", "vocab", "k", "ld_logits", "ld_grad")] + [
        (n, ctypes.c_void_p) for n in ("logits", "teacher_logits", "teacher_indices", "labels", "grad_loss")] + [
        (n, ctypes.c_double) for n in ("temperature", "label_weight", "grad_value")] + [
        (n, ctypes.c_int) for n in ("logits_dtype", "teacher_dtype", "index_bytes")] + [
        (n, ctypes.c_void_p) for n in ("loss", "stats", "grad")]


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 31), "vocab"),
    (dict(k=0), "k must"), (dict(k=1025), "k must"), (dict(logits_dtype=7), "dtypes"),
    (dict(index_bytes=2), "indices"), (dict(temperature=-1.0), "temperature"),
    (dict(label_weight=2.0), "label_weight"), (dict(logits=None), "null"),
    (dict(ld_logits=9), "overlap"), (dict(ld_grad=9), "overlap"),
    (dict(grad=(1 << 20) + 4), "overlap"), (dict(grad=1 << 20, ld_grad=11), "overlap"),
    (dict(loss=None), "null output"),
])
def test_distill_entry_checks_before_any_launch(change, message):
    lib = capi.load()
    base = dict(rows=4, vocab=10, k=3, ld_logits=10, ld_grad=10, logits=1 << 20,
                teacher_logits=1 << 21, teacher_indices=1 << 22, temperature=1.0, index_bytes=4,
                loss=1 << 23, grad=1 << 24)
    args = DistillArgs(**{**base, **change})
    assert lib.muon_train_distill_forward(ctypes.byref(args), None) == capi.ERR_INVALID_ARGUMENT
    assert message in capi.last_error()
    no_stats = DistillArgs(**base)
    assert lib.muon_train_distill_backward(ctypes.byref(no_stats), None) == capi.ERR_INVALID_ARGUMENT
    assert lib.muon_train_distill_forward(None, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.muon_train_distill_forward(ctypes.byref(DistillArgs(**{**base, "rows": 0})), None) == capi.OK


# ---------------------------------------------------------------------------------- fp8
F8 = torch.float8_e4m3fn


def test_fp8_blocks_refuses():
    with FakeTensorMode():
        ok = _cuda(200, 384, dtype=F8), _cuda(2, 3)
        assert train.Fp8Blocks(*ok).shape == (200, 384)
        assert train.Fp8Blocks(*ok, (200, 300)).shape == (200, 300)
        assert train.Fp8Blocks(ok[0], _cuda(200, 3)).shape == (200, 384)
        for bad, error in ((dict(values=_cuda(200, 384)), TypeError),
                           (dict(values=torch.zeros(200, 384).to(F8)), ValueError),
                           (dict(values=_cuda(384, dtype=F8)), ValueError),
                           (dict(values=_cuda(200, 0, dtype=F8)), ValueError),
                           (dict(scales=_cuda(2, 3, dtype=B16)), TypeError),
                           (dict(scales=_cuda(3, 3)), ValueError),
                           (dict(scales=_cuda(2, 4)), ValueError),
                           (dict(shape=(199, 384)), ValueError),
                           (dict(shape=(200, 200)), ValueError)):
            args = dict(values=ok[0], scales=ok[1])
            args.update(bad)
            with pytest.raises(error):
                train.Fp8Blocks(**args)


def test_fp8_calls_refuse_and_fake():
    with FakeTensorMode():
        x, w = _cuda(2, 3, 300, dtype=B16), _cuda(130, 300)
        q = train.quantize_fp8(w, 128)
        assert q.values.shape == (130, 384) and q.scales.shape == (2, 3) and q.shape == (130, 300)
        r = train.quantize_fp8(w)
        assert r.scales.shape == (130, 3) and r.scales.stride() == (1, 130)
        for call, error, message in (
                (lambda: train.quantize_fp8(_cuda(3)), ValueError, "shape"),
                (lambda: train.quantize_fp8(_cuda(3, 0)), ValueError, "shape"),
                (lambda: train.quantize_fp8(w, 64), ValueError, "block_rows"),
                (lambda: train.quantize_fp8(_cuda(3, 4, dtype=torch.float16)), TypeError, "x must"),
                (lambda: train.quantize_fp8(torch.zeros(3, 4)), ValueError, "ROCm GPU"),
                (lambda: train.fp8_matmul(w, q), TypeError, "Fp8Blocks"),
                (lambda: train.fp8_matmul(q, train.quantize_fp8(_cuda(9, 301))), ValueError, "width"),
                (lambda: train.fp8_matmul(q, r, torch.float16), TypeError, "dtype"),
                (lambda: train.fp8_linear(3.0, w), TypeError, "x must"),
                (lambda: train.fp8_linear(_cuda(), w), ValueError, "shape"),
                (lambda: train.fp8_linear(x, _cuda(130, 301)), ValueError, "weight"),
                (lambda: train.fp8_linear(x, _cuda(0, 300)), ValueError, "positive"),
                (lambda: train.fp8_linear(x, w.half()), TypeError, "weight"),
                (lambda: train.fp8_linear(_cuda(2, 301), q), ValueError, "columns"),
                (lambda: train.fp8_linear(_cuda(2, 300).requires_grad_(True), q), ValueError, "gradient")):
            with pytest.raises(error, match=message):
                call()
        assert train.fp8_matmul(r, q).shape == (130, 130)
        y = train.fp8_linear(x, q)
        assert y.shape == (2, 3, 130) and y.dtype == B16
        y = train.fp8_linear(x, w.requires_grad_(True))
        assert y.shape == (2, 3, 130) and y.requires_grad
        ops = torch.ops.muon_ascend950
        _, *saved = ops.fp8_linear_forward(x, w, 3)
        # x along 6 tokens, the weight along 130 rows: values, then scales
        assert saved[0].shape == (300 * 128 + 4 * 300,) and saved[1].shape == (300 * 256 + 4 * 2 * 3,)
        dx, dw = ops.fp8_linear_backward(y, *saved, 300, F32, 3)
        assert dx.shape == x.shape and dx.dtype == B16 and dw.shape == w.shape and dw.dtype == F32


class QuantizeArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("rows", "cols", "ld_x")] + [("x", ctypes.c_void_p)] + [
        (n, ctypes.c_int) for n in ("x_dtype", "block_rows")] + [
        (n, ctypes.c_void_p) for n in ("values", "scales", "values_t", "scales_t")]


class Operand(ctypes.Structure):
    _fields_ = [("values", ctypes.c_void_p), ("scales", ctypes.c_void_p)] + [
        (n, ctypes.c_int64) for n in ("ld", "scale_row", "scale_col")] + [("block_rows", ctypes.c_int)]


class MatmulArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("m", "n", "k")] + [("a", Operand), ("b", Operand),
                ("c", ctypes.c_void_p), ("ldc", ctypes.c_int64), ("c_dtype", ctypes.c_int)]


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows"), (dict(cols=1 << 31), "cols"), (dict(x_dtype=3), "dtype"),
    (dict(block_rows=64), "block_rows"), (dict(x=None), "null"), (dict(values=None), "null"),
    (dict(scales=None), "null"), (dict(values_t=4096), "null"), (dict(ld_x=9), "overlap"),
    (dict(values=4100), "aligned"), (dict(x=(1 << 21) + 16), "overlap"), (dict(rows=1 << 30, cols=1 << 30, ld_x=1 << 30), "too large"),
])
def test_quantize_entry_checks_before_any_launch(change, message):
    lib = capi.load()
    base = dict(rows=4, cols=10, ld_x=10, x=1 << 20, block_rows=1, values=1 << 21, scales=1 << 22)
    args = QuantizeArgs(**{**base, **change})
    assert lib.muon_train_fp8_quantize(ctypes.byref(args), None) == capi.ERR_INVALID_ARGUMENT
    assert message in capi.last_error()
    assert lib.muon_train_fp8_quantize(None, None) == capi.ERR_INVALID_ARGUMENT
    for empty in ("rows", "cols"):
        args = QuantizeArgs(**{**base, empty: 0})
        assert lib.muon_train_fp8_quantize(ctypes.byref(args), None) == capi.OK


@pytest.mark.parametrize("change,operand,message", [
    (dict(m=-1), {}, "m, n and k"), (dict(k=100), {}, "multiple of 128"), (dict(c=None), {}, "null"),
    (dict(c_dtype=2), {}, "dtype"), (dict(ldc=7), {}, "overlap"), ({}, dict(values=None), "null"),
    ({}, dict(scales=None), "null"), ({}, dict(values=4104), "aligned"), ({}, dict(ld=264), "aligned"),
    ({}, dict(ld=128), "overlap"), ({}, dict(ld=1 << 23), "far apart"),
    ({}, dict(block_rows=2), "block_rows"), ({}, dict(scale_row=2), "next to each other"),
    ({}, dict(scale_row=1 << 27), "far apart"), ({}, dict(scale_col=1 << 28), "far apart"),
    (dict(c=(1 << 20) + 128), {}, "overlap"),
    (dict(m=1 << 30, n=1 << 30, ldc=1 << 30), {}, None),
])
def test_matmul_entry_checks_before_any_launch(change, operand, message):
    lib = capi.load()
    good = dict(values=1 << 20, scales=1 << 22, ld=256, scale_row=1, scale_col=4, block_rows=1)
    base = dict(m=4, n=8, k=256, c=1 << 24, ldc=8)
    args = MatmulArgs(**{**base, **change}, a=Operand(**{**good, **operand}), b=Operand(**good))
    status = lib.muon_train_fp8_matmul(ctypes.byref(args), None)
    if message is None:  # too large, or no device to say for
        assert status in (capi.ERR_INVALID_ARGUMENT, capi.ERR_HIP)
    else:
        assert status == capi.ERR_INVALID_ARGUMENT and message in capi.last_error()
    for empty in ("m", "n"):
        args = MatmulArgs(**{**base, empty: 0}, a=Operand(**good), b=Operand(**good))
        assert lib.muon_train_fp8_matmul(ctypes.byref(args), None) == capi.OK


class DecodeArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("m", "n", "cols", "ld_x")] + [
        ("x", ctypes.c_void_p), ("x_dtype", ctypes.c_int), ("w", Operand), ("c", ctypes.c_void_p),
        ("ldc", ctypes.c_int64), ("c_dtype", ctypes.c_int)]


@pytest.mark.parametrize("change,operand,message", [
    (dict(m=17), {}, "m must"), (dict(m=-1), {}, "m must"), (dict(cols=0), {}, "cols"),
    (dict(x_dtype=2), {}, "dtype"), (dict(x=None), {}, "null"), (dict(c=None), {}, "null"),
    (dict(ld_x=199), {}, "overlap"), (dict(ldc=7), {}, "overlap"),
    ({}, dict(ld=128), "overlap"), ({}, dict(values=4104), "aligned"),
    ({}, dict(block_rows=1), "block_rows"), (dict(c=(1 << 23) - 4), {}, "overlap"),
    (dict(x=(1 << 24) + 4), {}, "overlap"),
])
def test_decode_entry_checks_before_any_launch(change, operand, message):
    lib = capi.load()
    good = dict(values=1 << 20, scales=1 << 22, ld=256, scale_row=1, scale_col=4, block_rows=128)
    base = dict(m=4, n=8, cols=200, ld_x=200, x=1 << 23, c=1 << 24, ldc=8)
    args = DecodeArgs(**{**base, **change}, w=Operand(**{**good, **operand}))
    assert lib.muon_train_fp8_decode(ctypes.byref(args), None) == capi.ERR_INVALID_ARGUMENT
    assert message in capi.last_error()
    assert lib.muon_train_fp8_decode(None, None) == capi.ERR_INVALID_ARGUMENT
    for empty in ("m", "n"):
        args = DecodeArgs(**{**base, empty: 0}, w=Operand(**good))
        assert lib.muon_train_fp8_decode(ctypes.byref(args), None) == capi.OK


def test_missing_tensors_are_named():
    with FakeTensorMode():
        for call, name in ((lambda: train.block_norms(None, _cuda(2, 8)), "y"),
                           (lambda: train.distill_topk(_cuda(2, 8), None, _cuda(2, 1, dtype=torch.int64)),
                            "teacher_logits"),
                           (lambda: train.fp8_linear(None, _cuda(2, 8)), "x"),
                           (lambda: train.fp8_linear(_cuda(2, 8), 3.0), "weight")):
            with pytest.raises(TypeError, match=name):
                call()


def test_matmul_workspace_entry():
    lib = capi.load()
    good = dict(values=1 << 20, scales=1 << 22, ld=256, scale_row=1, scale_col=4, block_rows=1)
    args = MatmulArgs(m=4, n=8, k=256, c=1 << 24, ldc=8, a=Operand(**good), b=Operand(**good))
    size = ctypes.c_size_t(7)
    assert lib.muon_train_fp8_matmul_workspace(None, ctypes.byref(size)) == capi.ERR_INVALID_ARGUMENT
    assert lib.muon_train_fp8_matmul_workspace(ctypes.byref(args), None) == capi.ERR_INVALID_ARGUMENT
    assert lib.muon_train_fp8_matmul_in(None, None, ctypes.c_size_t(0), None) == capi.ERR_INVALID_ARGUMENT
    odd = ctypes.c_void_p((1 << 26) + 8)
    assert lib.muon_train_fp8_matmul_in(ctypes.byref(args), odd, ctypes.c_size_t(64), None) == capi.ERR_INVALID_ARGUMENT
    assert "aligned" in capi.last_error()
    args.m = -1
    assert lib.muon_train_fp8_matmul_workspace(ctypes.byref(args), ctypes.byref(size)) == capi.ERR_INVALID_ARGUMENT
    assert size.value == 0
    args.m = 0
    assert lib.muon_train_fp8_matmul_workspace(ctypes.byref(args), ctypes.byref(size)) == capi.OK and size.value == 0
    assert lib.muon_train_fp8_matmul_in(ctypes.byref(args), None, ctypes.c_size_t(0), None) == capi.OK


@pytest.mark.parametrize("temperature", [1e-39, 1e-46, 5e-324, 1e30])
def test_distill_refuses_temperatures_that_float32_does_not_hold(temperature):
    """1 / temperature has to be finite in float32."""
    with FakeTensorMode():
        for call in (train.distill_topk, train.distill_topk_with_grad):
            args, kw = _distill_ok(temperature=temperature)
            with pytest.raises(ValueError, match="temperature"):
                call(*args, **kw)
        args, kw = _distill_ok(temperature=1.2e-38)
        train.distill_topk(*args, **kw)
    args = DistillArgs(rows=4, vocab=10, k=3, ld_logits=10, ld_grad=10, logits=1 << 20,
                       teacher_logits=1 << 21, teacher_indices=1 << 22, temperature=temperature,
                       index_bytes=4, loss=1 << 23)
    assert capi.load().muon_train_distill_forward(ctypes.byref(args), None) == capi.ERR_INVALID_ARGUMENT
    assert "temperature" in capi.last_error()


# ------------------------------------------------------------------------ forward mode
def _forward_mode_calls():
    """Each public call on one differentiable operand, by name."""
    def index():
        return _cuda(4, 3, dtype=torch.int64)

    return {
        "norms y": lambda x: train.block_norms(x, _cuda(4, 64))[0],
        "norms residual": lambda x: train.block_norms(_cuda(4, 64), x)[0],
        "norms gate": lambda x: train.block_norms(_cuda(4, 64), _cuda(4, 64), gate=x)[0],
        "norms weight": lambda x: train.block_norms(_cuda(4, 64), _cuda(4, 64), post_weight=x[0])[0],
        "norms scale": lambda x: train.block_norms(_cuda(4, 64), _cuda(4, 64), residual_scale=x[0])[0],
        "distill logits": lambda x: train.distill_topk(x, _cuda(4, 3), index()),
        "distill teacher": lambda x: train.distill_topk(_cuda(4, 64), x[:, :3], index()),
        "with_grad logits": lambda x: train.distill_topk_with_grad(x, _cuda(4, 3), index())[1],
        "with_grad weight": lambda x: train.distill_topk_with_grad(
            _cuda(4, 64), _cuda(4, 3), index(), grad_loss=x[:, 0])[1],
        "linear x": lambda x: train.fp8_linear(x, _cuda(8, 64)),
        "linear weight": lambda x: train.fp8_linear(_cuda(5, 64), x),
        "serving x": lambda x: train.fp8_linear(x, train.quantize_fp8(_cuda(8, 64), 128)),
    }


@pytest.mark.parametrize("name", _forward_mode_calls())
def test_forward_mode_is_refused(name):
    """No operator has a forward-mode derivative; a tangent is refused, never dropped."""
    import torch.autograd.forward_ad as fwd

    call = _forward_mode_calls()[name]
    with FakeTensorMode():
        with fwd.dual_level():
            x = fwd.make_dual(_cuda(4, 64), _cuda(4, 64))
            with pytest.raises(NotImplementedError, match="forward"):
                call(x)
            call(_cuda(4, 64))  # without a tangent nothing is refused
        x, t = _cuda(4, 64), _cuda(4, 64)
        with pytest.raises(NotImplementedError, match="forward"):
            torch.func.jvp(call, (x,), (t,))
        if "with_grad" not in name:  # writes into a tensor: no vmap
            with pytest.raises(NotImplementedError, match="forward"):
                torch.func.jvp(torch.vmap(call), (_cuda(2, 4, 64),), (_cuda(2, 4, 64),))


@pytest.mark.parametrize("tokens,n,k,wanted", [
    ((1 << 22) + 1, 64, 64, "weight"),  # a row of the transposed operands
    (1 << 21, 64, 1 << 14, "weight"), (1 << 21, 1 << 14, 64, "weight"),  # their scales
    (1 << 21, 1 << 14, 64, "x"),  # the gradient's scales
])
def test_fp8_linear_refuses_what_its_backward_pass_could_not_do(tokens, n, k, wanted):
    """At the call, not in the backward pass that follows it."""
    with FakeTensorMode():
        x, w = _cuda(tokens, k, dtype=B16), _cuda(n, k)
        train.fp8_linear(x, w)  # no gradient wanted
        (w if wanted == "weight" else x).requires_grad_(True)
        with pytest.raises(ValueError, match="tokens"):
            train.fp8_linear(x, w)
        with torch.no_grad():
            train.fp8_linear(x, w)
        less = x[: 1 << 14]
        assert train.fp8_linear(less, w).requires_grad
