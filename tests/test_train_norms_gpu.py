"""block_norms on the GPU against its formula in 64 bits: shapes from one channel to the
widest rows, every kind of gate and scale, both dtypes of each operand, strides, empty
inputs, rows of zeros and of infinities, gradients against the formula's and against
differences."""

from __future__ import annotations

import pytest
import torch

import muon_fusion_ascend950_amd as mf
from tests.train_checks import F32_ROW, F32_SUM, check, leaf, randn

pytestmark = pytest.mark.gpu
F32, B16 = torch.float32, torch.bfloat16
EPS = 1e-6


def formula(y, residual, post_weight, gate, scale, pre_weight, post_norm, pre_norm, eps=EPS):
    """In the arithmetic of its inputs; returns (residual_out, normed)."""
    def norm(x):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)

    u = norm(y) if post_norm else y
    if post_weight is not None:
        u = u * post_weight
    total = residual * scale + (u if gate is None else u * gate)
    if not pre_norm:
        return total, None
    h = norm(total)
    return total, h if pre_weight is None else h * pre_weight


def make(shape, ty=F32, tr=F32, tw=F32, gate="channel", scale="number", weights=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    d = shape[-1]
    gate_shape = {"none": None, "channel": (d,), "token": (*shape[:-1], 1), "full": shape,
                  "sequence": (shape[0],) + (1,) * (len(shape) - 2) + (d,)}[gate]
    tg = F32 if gate == "channel" else ty
    t = dict(
        y=randn(gen, *shape, dtype=ty), residual=randn(gen, *shape, dtype=tr, scale=3.0),
        post_weight=(1 + randn(gen, d, scale=0.2)).to(tw) if weights else None,
        gate=None if gate_shape is None else randn(gen, *gate_shape).to(tg),
        scale={"number": 0.9, "scalar": 0.9 + randn(gen, 1, scale=0.1),
               "vector": 0.9 + randn(gen, d, scale=0.1)}[scale],
        pre_weight=(1 + randn(gen, d, scale=0.2)).to(tw) if weights else None)
    t = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in t.items()}
    grads = (randn(gen, *shape, dtype=tr).cuda(), randn(gen, *shape, dtype=ty).cuda())
    return t, grads


def call(t, post_norm=True, pre_norm=True):
    return mf.train.block_norms(t["y"], t["residual"], post_weight=t["post_weight"],
                                gate=t["gate"], residual_scale=t["scale"],
                                pre_weight=t["pre_weight"], post_norm=post_norm,
                                pre_norm=pre_norm, eps=EPS)


def run_both(t, grads, post_norm=True, pre_norm=True):
    """Checks both outputs and the gradients of every tensor."""
    names = [k for k, v in t.items() if isinstance(v, torch.Tensor)]
    for k in names:
        t[k].requires_grad_(True)
    exact = {k: leaf(v) for k, v in t.items()}
    want = formula(*(exact[k] for k in ("y", "residual", "post_weight", "gate", "scale", "pre_weight")),
                   post_norm, pre_norm)
    got = call(t, post_norm, pre_norm)
    assert got[0].dtype == t["residual"].dtype
    check(got[0], want[0], F32_ROW, "residual_out")
    if not pre_norm:
        assert got[1] is None
        got, want, grads = got[:1], want[:1], grads[:1]
    else:
        assert got[1].dtype == t["y"].dtype
        check(got[1], want[1], F32_ROW, "normed")
    with torch.no_grad():  # the same without a gradient to follow
        again = call(t, post_norm, pre_norm)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    mine = torch.autograd.grad(got, [t[k] for k in names], grads)
    theirs = torch.autograd.grad(want, [exact[k] for k in names], [g.double() for g in grads])
    for k, a, b in zip(names, mine, theirs):
        assert a.dtype == t[k].dtype and a.shape == t[k].shape
        rows = k in ("y", "residual") or a.shape == t["y"].shape
        check(a, b, F32_ROW if rows else F32_SUM, "gradient of " + k)


SHAPES = [(1, 1, 1), (1, 1, 7), (2, 3, 8), (1, 3, 129), (3, 5, 513), (2, 33, 768), (1, 1, 1025),
          (7, 41, 2051), (2, 300, 2048), (1, 1, 4096), (3, 67, 4100), (1, 9, 8200), (2, 3, 16384)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("ty,tr", [(B16, B16), (B16, F32), (F32, F32), (F32, B16)], ids=str)
def test_shapes_and_dtypes(shape, ty, tr):
    run_both(*make(shape, ty, tr))


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token", "full"])
@pytest.mark.parametrize("scale", ["number", "scalar", "vector"])
@pytest.mark.parametrize("shape", [(3, 70, 515), (5, 2, 1024)], ids=str)
def test_gates_and_scales(shape, gate, scale):
    run_both(*make(shape, B16, F32, gate=gate, scale=scale))


@pytest.mark.parametrize("gate", ["sequence", "token", "full"])
def test_many_sequences_and_rows(gate):
    # more sequences than workgroups stay resident, and more rows than workgroups
    run_both(*make((3000, 3, 72), F32, F32, gate=gate, scale="scalar"))
    run_both(*make((1, 5000, 200), F32, F32, gate=gate, scale="vector"))


@pytest.mark.parametrize("gate,scale", [("full", "number"), ("token", "vector"), ("sequence", "scalar")])
@pytest.mark.parametrize("ty,tr", [(B16, B16), (F32, F32)], ids=str)
@pytest.mark.parametrize("shape", [(2, 300, 1500), (2, 290, 3001), (1, 270, 5120), (2, 140, 9000)], ids=str)
def test_gates_of_wide_rows(shape, ty, tr, gate, scale):
    """Each number of threads and pieces of a row, several rows a workgroup."""
    run_both(*make(shape, ty, tr, gate=gate, scale=scale))


def test_gate_over_several_axes():
    run_both(*make((2, 3, 4, 96), F32, F32, gate="sequence"))
    run_both(*make((11, 96), F32, F32, gate="token"))
    t, grads = make((11, 96), F32, F32, gate="none")
    t["gate"] = torch.full((1, 96), 0.5, device="cuda")
    run_both(t, grads)


@pytest.mark.parametrize("post_norm,pre_norm", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("gate", ["none", "token"])
def test_norms_left_out(post_norm, pre_norm, gate):
    t, grads = make((2, 19, 300), B16, F32, gate=gate, scale="vector")
    if not pre_norm:
        t["pre_weight"] = None
    run_both(t, grads, post_norm, pre_norm)


@pytest.mark.parametrize("tw", [F32, B16], ids=str)
def test_weight_dtypes_and_no_weights(tw):
    run_both(*make((2, 40, 640), B16, B16, tw=tw))
    run_both(*make((2, 40, 640), B16, B16, weights=False, gate="none"))


def test_strides_and_offsets():
    base, grads = make((6, 50, 2 * 96 + 3), F32, F32, gate="none", weights=False)
    cut = {"y": base["y"][:, :, 3:99], "residual": base["residual"][:, 1::2, 1:97]}
    t = dict(base, y=cut["y"][:, ::2], residual=cut["residual"])  # rows apart, unaligned
    g = tuple(x[:, :25, :96] for x in grads)
    run_both({k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in t.items()}, g)
    t = dict(base, y=base["y"].mT, residual=base["residual"].mT)  # columns apart
    run_both({k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in t.items()},
             tuple(x.mT for x in grads))
    one = torch.full((1, 1, 1), 0.25, device="cuda").expand(6, 25, 96)  # broadcast gradients
    t = {"y": torch.randn(6, 25, 96, device="cuda"), "residual": one * 4.0, "gate": None,
         "post_weight": None, "pre_weight": None, "scale": 1.0}
    run_both(t, (one, one))


def test_one_output_used():
    for used in (0, 1):
        t, grads = make((4, 30, 520), F32, F32, gate="full", scale="vector")
        exact = {k: leaf(v) for k, v in t.items()}
        names = [k for k in t if isinstance(t[k], torch.Tensor) and (used or k != "pre_weight")]
        for k in names:
            t[k].requires_grad_(True)
        args = ("y", "residual", "post_weight", "gate", "scale", "pre_weight")
        want = formula(*(exact[k] for k in args), True, True)[used]
        theirs = torch.autograd.grad(want, [exact[k] for k in names], grads[used].double())
        mine = torch.autograd.grad(call(t)[used], [t[k] for k in names], grads[used])
        for k, a, b in zip(names, mine, theirs):
            check(a, b, F32_SUM, "gradient of " + k)


def test_only_some_gradients_wanted():
    t, grads = make((4, 30, 520), F32, F32, gate="sequence", scale="vector")
    whole = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    every = dict(zip(whole, torch.autograd.grad(call(whole), list(whole.values()), grads)))
    for k in t:
        part = {n: v.detach().clone().requires_grad_(n == k) for n, v in t.items()}
        (g,) = torch.autograd.grad(call(part), [part[k]], grads)
        assert torch.equal(g, every[k]), k


def test_empty_inputs():
    t, _ = make((1, 1, 64), F32, F32)
    y = torch.empty(0, 5, 64, device="cuda", requires_grad=True)
    w = t["post_weight"].requires_grad_(True)
    out, h = mf.train.block_norms(y, y.detach(), post_weight=w, gate=t["gate"])
    assert out.shape == h.shape == (0, 5, 64)
    (out.sum() + h.sum()).backward()
    assert y.grad.shape == y.shape and torch.equal(w.grad, torch.zeros_like(w))


def test_rows_keep_to_themselves():
    """A row of zeros gives finite results, and a row with an infinity or a NaN touches
    only itself."""
    t, _ = make((1, 9, 300), B16, F32, gate="channel")
    clean = call(t)
    t["y"][0, 2] = 0.0
    t["residual"][0, 2] = 0.0
    t["y"][0, 4, 17] = float("inf")
    t["residual"][0, 6, 299] = float("nan")
    out, h = call(t)
    rows = [0, 1, 3, 5, 7, 8]
    assert torch.equal(out[:, rows], clean[0][:, rows]) and torch.equal(h[:, rows], clean[1][:, rows])
    assert torch.equal(out[0, 2], torch.zeros_like(out[0, 2]))
    assert torch.equal(h[0, 2], torch.zeros_like(h[0, 2]))
    assert h[0, 6].isnan().all() and out[0, 6, :299].isfinite().all()


def test_same_bits_every_run_and_on_another_stream():
    t, grads = make((2, 700, 1030), B16, B16, gate="sequence", scale="scalar")
    for v in t.values():
        v.requires_grad_(True)

    def once():
        out = call(t)
        return (*out, *torch.autograd.grad(out, list(t.values()), grads))

    first = once()
    assert all(torch.equal(a, b) for a, b in zip(first, once()))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = once()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_gradient_against_differences():
    """The loss <out, a> + <h, b> along a random direction, central differences with step h:
    its truncation error is about h² of the third derivative, and float32 outputs of size 1
    to 10 leave about 1e-7 / h of noise in each term, averaged over 10 000 of them; both
    stay under 1e-3 of the slope at h = 1/64."""
    t, grads = make((2, 25, 200), F32, F32, gate="sequence", scale="vector", seed=3)
    names = list(t)
    for k in names:
        t[k].requires_grad_(True)

    def loss(v):
        return sum((o.double() * g.double()).sum() for o, g in zip(call(v), grads))

    slopes = torch.autograd.grad(loss(t), [t[k] for k in names])
    gen = torch.Generator().manual_seed(5)
    h = 1.0 / 64
    for k, g in zip(names, slopes):
        way = randn(gen, *t[k].shape).cuda()
        with torch.no_grad():
            up = loss({**t, k: t[k] + h * way})
            down = loss({**t, k: t[k] - h * way})
        slope = (g.double() * way.double()).sum()
        size = (g.double().norm() * way.double().norm()) / way.numel() ** 0.5
        assert abs((up - down) / (2 * h) - slope) <= 1e-3 * size, k


def test_captured_in_a_graph():
    t, grads = make((1, 130, 515), B16, B16, gate="channel", scale="scalar")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        call(t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        held = call(t)
    for seed in range(3):
        new, _ = make((1, 130, 515), B16, B16, gate="channel", scale="scalar", seed=seed + 10)
        with torch.no_grad():
            for k in t:
                t[k].copy_(new[k])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, call(new)))


@pytest.mark.parametrize("shape", [(3, 0, 40), (2, 5, 0, 40), (0, 4, 40)], ids=str)
def test_sequences_without_tokens(shape):
    """A gate vector for each sequence of none: nothing comes out, its gradient is zero."""
    y, r = (torch.empty(shape, device="cuda", requires_grad=True) for _ in range(2))
    gate = torch.ones(shape[0], *(1 for _ in shape[1:-1]), 40, device="cuda", requires_grad=True)
    weight = torch.ones(40, device="cuda", requires_grad=True)
    with torch.no_grad():
        out, h = mf.train.block_norms(y, r, gate=gate, post_weight=weight)
    assert out.shape == h.shape == shape
    out, h = mf.train.block_norms(y, r, gate=gate, post_weight=weight)
    (out.sum() + h.sum()).backward()
    for t in (y, r, gate, weight):
        assert t.grad.shape == t.shape and not t.grad.any()


def test_more_sequences_than_a_launch_takes():
    """A launch has at most 2^32 - 1 threads, a sequence with a gate of its own 64 of them."""
    b = (1 << 26) + 3
    gen = torch.Generator(device="cuda").manual_seed(1)
    # two tokens of one channel that is left as it is: each gradient is a product or a sum of two
    y, r = (torch.randint(-4, 5, (b, 2, 1), device="cuda", generator=gen).bfloat16() for _ in range(2))
    gate = torch.randint(1, 5, (b, 1, 1), device="cuda", generator=gen).bfloat16()
    d_out = torch.randint(-2, 3, (b, 2, 1), device="cuda", generator=gen).bfloat16()
    leaves = [t.requires_grad_(True) for t in (y, r, gate)]
    out, _ = mf.train.block_norms(y, r, gate=gate, post_norm=False, pre_norm=False)
    dy, dr, dgate = torch.autograd.grad(out, leaves, d_out)
    assert torch.equal(out, r + gate * y) and torch.equal(dr, d_out)
    assert torch.equal(dy, gate * d_out)
    assert torch.equal(dgate, (d_out * y).sum(1, keepdim=True))
