"""The training-step operators together on the GPU: the example's student learns, and a block
of them traced by torch.compile gives eager's bits."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from muon_fusion_ascend950_amd import train

pytestmark = pytest.mark.gpu


def test_example_student_learns():
    path = Path(__file__).resolve().parent.parent / "examples" / "distill_step.py"
    spec = importlib.util.spec_from_file_location("distill_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, _ = example.train(30, width=256, layers=2)
    # a random vocabulary of 4099 with 16 entries: the student starts near log(4099) plus its
    # own logits' spread, and memorises some of 1024 fixed tokens within a few steps
    assert all(later < losses[0] for later in losses[5:]) and losses[-1] < 0.9 * losses[0], losses
    again, _ = example.train(3, width=256, layers=2)
    assert again == losses[:3]  # the same bits every run


def test_traced_step_equals_eager():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(2, 33, 160, generator=gen).cuda()
    y = torch.randn(2, 33, 160, generator=gen).to(torch.bfloat16).cuda()
    w = torch.randn(300, 160, generator=gen).cuda()
    post, scale = torch.ones(160).cuda(), torch.ones(1).cuda()
    teacher = torch.randn(2, 33, 4, generator=gen).cuda()
    index = torch.randint(0, 300, (2, 33, 4), generator=gen).cuda()

    def step(x, y, w, post, scale):
        r, h = train.block_norms(y, x, post_weight=post, residual_scale=scale)
        loss = train.distill_topk(train.fp8_linear(h, w), teacher, index, temperature=2.0)
        return loss.sum() + r.float().square().sum()

    def run(f):
        args = [t.detach().clone().requires_grad_(True) for t in (x, y, w, post, scale)]
        out = f(*args)
        return [out, *torch.autograd.grad(out, args)]

    torch._dynamo.reset()
    want = run(step)
    got = run(torch.compile(step, backend="aot_eager", fullgraph=True))
    # the sums around the operators are torch's and may be fused differently: none is here
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_have_none_of_their_own():
    """A pass that keeps its graph gives the same gradients; differentiating them is refused."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(20, 160, generator=gen).cuda().requires_grad_(True)
    w = torch.randn(130, 160, generator=gen).cuda().requires_grad_(True)
    teacher = torch.randn(20, 3, generator=gen).cuda()
    index = torch.randint(0, 130, (20, 3), generator=gen).cuda()
    for out in (train.block_norms(x, x, gate=w[0])[1].sum(), train.fp8_linear(x, w).sum(),
                train.distill_topk(x, teacher, index).sum()):
        (plain,) = torch.autograd.grad(out, x, retain_graph=True)
        (kept,) = torch.autograd.grad(out, x, create_graph=True)
        assert torch.equal(plain, kept)
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            kept.sum().backward()


def test_a_gradient_has_no_forward_mode_derivative():
    """Differentiating a backward pass in forward mode is refused, not answered with zeros."""
    import torch.autograd.forward_ad as fwd

    gen = torch.Generator().manual_seed(2)
    x = torch.randn(20, 160, generator=gen).cuda().requires_grad_(True)
    w = torch.randn(130, 160, generator=gen).cuda()
    teacher = torch.randn(20, 3, generator=gen).cuda()
    index = torch.randint(0, 130, (20, 3), generator=gen).cuda()
    for out in (train.block_norms(x, x)[1], train.fp8_linear(x, w), train.distill_topk(x, teacher, index)):
        with fwd.dual_level():
            grad = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(out, x, grad, retain_graph=True)
        torch.autograd.grad(out, x, torch.ones_like(out))


def test_an_error_of_an_earlier_call_is_not_the_operators():
    """An error that another HIP call of this thread left behind is its caller's to read: the
    operators report what became of their own launches."""
    import ctypes

    gen = torch.Generator().manual_seed(3)
    x = torch.randn(40, 256, generator=gen).cuda()
    w = torch.randn(300, 256, generator=gen).cuda()
    teacher = torch.randn(40, 3, generator=gen).cuda()
    index = torch.randint(0, 256, (40, 3), generator=gen).cuda()
    weight = train.quantize_fp8(w, 128)
    calls = [lambda: train.quantize_fp8(x), lambda: train.fp8_linear(x, weight), lambda: train.fp8_linear(x[:2], weight),
             lambda: train.fp8_linear(x, w), lambda: train.block_norms(x, x),
             lambda: train.distill_topk(x, teacher, index), lambda: train.distill_topk_with_grad(x, teacher, index)]
    for call in calls:
        call()
    with open("/proc/self/maps") as maps:
        hip = ctypes.CDLL(next(line.split()[-1] for line in maps if "libamdhip64.so" in line))
    try:
        for call in calls:
            assert hip.hipSetDevice(1 << 20) != 0
            call()
    finally:
        hip.hipGetLastError()
