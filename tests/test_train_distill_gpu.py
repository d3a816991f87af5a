"""distill_topk and distill_topk_with_grad on the GPU against the formula in 64 bits:
vocabularies from one entry to past what registers hold, odd ones, every entry count,
absent entries and rows, repeated indices, masked and extreme logits, labels, strides, the
gradient in place, and the gradient against differences.

Tolerances (2-norms, see train_checks): the loss sums K terms of size up to about
max(1, |log q|) whose errors are a few 2^-24 of that, while the loss itself may be smaller:
1e-5 of the losses' norm.  A float32 gradient element q - p has an error of a few 2^-24 of q
and of the exponent's argument, |x| * 2^-24 * 1.44 relative, |x| up to 30: 1e-5."""

from __future__ import annotations

import math

import pytest
import torch

import muon_fusion_ascend950_amd as mf
from tests.train_checks import check, randn

pytestmark = pytest.mark.gpu
F32, B16 = torch.float32, torch.bfloat16
BOUND = 1e-5


def formula(z, teacher, index, tau, labels, lam, weight):
    """(loss, gradient of sum(weight * loss)) in float64."""
    z = z.detach().double()
    v = z.shape[-1]
    present = (index >= 0) & (index < v)
    at = torch.where(present, index, 0).long()
    t = torch.where(present, teacher.double() / tau, -math.inf)
    some = (t > -math.inf).any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, t, 0.0), -1), 0.0)
    p = torch.where(present, p, 0.0)
    log_q = torch.log_softmax(z / tau, -1)
    terms = torch.where(p > 0, p * (torch.log(p) - log_q.gather(-1, at)), 0.0)
    loss = (1 - lam) * tau * tau * terms.sum(-1)
    grad = (1 - lam) * tau * torch.where(some, torch.exp(log_q), 0.0)
    grad = grad.scatter_add(-1, at, -(1 - lam) * tau * p)
    if labels is not None:
        known = (labels >= 0) & (labels < v)
        safe = torch.where(known, labels, 0)
        hard = torch.log_softmax(z, -1)
        loss = loss - lam * torch.where(known, hard.gather(-1, safe[..., None])[..., 0], 0.0)
        ce = torch.exp(hard).scatter_add(-1, safe[..., None], -torch.ones_like(z[..., :1]))
        grad = grad + lam * torch.where(known[..., None], ce, 0.0)
    return loss, grad * weight.double()[..., None]


def make(rows, v, k, dtype=F32, teacher=F32, index=torch.int64, labels=False, absent=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    z = randn(gen, rows, v, scale=2.5)
    t = z + randn(gen, rows, v, scale=1.5)
    top, at = torch.topk(t, min(k, v), dim=1)
    if k > v:  # more entries than there are: absent ones
        at = torch.cat([at, torch.full((rows, k - v), -1)], 1)
        top = torch.cat([top, torch.full((rows, k - v), math.nan)], 1)
    if absent:
        count = torch.randint(0, k + 1, (rows, 1), generator=gen)
        gone = torch.arange(k) >= count
        at[gone] = -1
        top[gone] = math.nan  # never looked at
    y = torch.randint(0, v, (rows,), generator=gen)
    y[::3] = -100
    weight = torch.rand(rows, generator=gen) - 0.25
    return dict(z=z.to(dtype).cuda(), teacher=top.to(teacher).cuda(), index=at.to(index).cuda(),
                labels=y.cuda() if labels else None, weight=weight.cuda())


def run_all(s, tau=1.0, lam=0.0, bound=BOUND):
    """The three forms against the formula; the two gradients have the same bits."""
    lam = lam if s["labels"] is not None else 0.0
    want = formula(s["z"], torch.nan_to_num(s["teacher"]) if s.get("nan_ok") else s["teacher"],
                   s["index"], tau, s["labels"], lam, s["weight"])
    kw = dict(temperature=tau, labels=s["labels"], label_weight=lam)
    args = (s["teacher"], s["index"])
    loss = mf.train.distill_topk(s["z"], *args, **kw)
    assert loss.dtype == F32
    check(loss, want[0], bound, "loss")
    one, grad = mf.train.distill_topk_with_grad(s["z"], *args, grad_loss=s["weight"], **kw)
    assert grad.dtype == s["z"].dtype and torch.equal(one.nan_to_num(), loss.nan_to_num())
    check(grad, want[1], bound, "gradient")
    z = s["z"].detach().clone().requires_grad_(True)
    (auto,) = torch.autograd.grad(mf.train.distill_topk(z, *args, **kw), z, s["weight"])
    assert torch.equal(auto.nan_to_num(), grad.nan_to_num())
    return loss, grad


@pytest.mark.parametrize("v", [1, 2, 7, 64, 129, 1000, 2049, 4096, 8195, 16390, 32768, 50001])
@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
def test_vocabularies(v, dtype):
    run_all(make(5, v, min(v, 13), dtype), tau=2.0)


@pytest.mark.parametrize("v,dtype", [(65536, F32), (65541, F32), (131072, B16), (200003, B16)], ids=str)
def test_rows_past_the_registers(v, dtype):
    run_all(make(3, v, 50, dtype, labels=True), tau=1.5, lam=0.3)


def test_the_largest_logit_past_the_registers():
    s = make(4, 140000, 4, F32)
    s["z"][0, 139999] = 60.0
    s["z"][1, 70000:] = -math.inf
    s["z"][2, :70000] = -math.inf
    s["index"][2] = torch.arange(100000, 100004)
    s["index"][1] = torch.arange(4)
    run_all(s)


@pytest.mark.parametrize("k", [1, 2, 64, 255, 256, 257, 700, 1024])
@pytest.mark.parametrize("labels", [False, True])
def test_entry_counts(k, labels):
    run_all(make(6, 3001, k, B16, B16, torch.int32, labels), tau=1.0, lam=0.5)
    run_all(make(3, 20011, k, F32, F32, torch.int64, labels), tau=3.0, lam=1.0)


@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
def test_absent_entries_and_rows(dtype):
    s = make(64, 777, 9, dtype, labels=True, absent=True)
    s["index"][5] = -1  # a row without entries: only the label's term
    s["labels"][5] = 3
    s["index"][6] = 777  # nor inside the vocabulary
    s["labels"][6] = -100  # and without a label: nothing at all
    s["labels"][8] = 777
    s["teacher"][7] = -math.inf  # entries without weight
    s["index"][7] = torch.arange(9)
    clean = dict(s, teacher=torch.where(s["index"] < 0, 0.0, s["teacher"]))
    loss, grad = run_all(clean, tau=1.0, lam=0.4)
    assert loss[6] == 0 and not grad[6].any()
    other, other_grad = mf.train.distill_topk_with_grad(
        s["z"], s["teacher"], s["index"], grad_loss=s["weight"], labels=s["labels"], label_weight=0.4)
    assert torch.equal(loss, other) and torch.equal(grad, other_grad)  # NaN never looked at


def test_more_entries_than_vocabulary():
    s = make(4, 5, 8, F32)
    s["teacher"] = s["teacher"].nan_to_num()
    run_all(s)


def test_an_index_that_occurs_twice():
    s = make(4, 100, 6, F32, labels=True)
    s["index"][0] = 17
    s["index"][1, 3] = s["index"][1, 0]
    s["labels"][1] = s["index"][1, 0]
    s["labels"][2] = s["index"][2, 2]
    run_all(s, tau=2.0, lam=0.5)


@pytest.mark.parametrize("k", [15, 16, 17, 100, 1024])
def test_indices_that_occur_often(k):
    """Each of an element's entries counts, wherever they stand among the others."""
    s = make(5, 3000, k, F32, labels=True, seed=k)
    gen = torch.Generator().manual_seed(k)
    s["index"][1:] = torch.randint(0, 6, (4, k), generator=gen).cuda() * 499
    s["labels"][2] = 499
    run_all(s, tau=2.0, lam=0.5)


@pytest.mark.parametrize("v,dtype", [(98304, F32), (98311, F32), (140000, F32), (131080, B16), (160001, B16)], ids=str)
def test_rows_in_registers_and_lds(v, dtype):
    run_all(make(3, v, 40, dtype, labels=True), tau=1.5, lam=0.3)


def test_masked_and_extreme_logits():
    s = make(8, 1003, 5, F32)
    s["z"][:, -3:] = -math.inf
    s["index"] = s["index"].clamp(max=990)
    s["z"][1, 500:] = torch.finfo(F32).min  # the type's lowest value
    s["z"][2] = torch.finfo(F32).min  # everywhere: a uniform row
    s["z"][3] *= 30.0  # one logit holds nearly all
    s["z"][4, 7] = 3e38
    s["index"][1] = torch.arange(5)
    s["index"][4, 0] = 7
    s["teacher"][5, 2] = -math.inf
    run_all(s, tau=0.5, bound=2e-5)  # arguments up to 1e39: exponents of the few that count
    low = make(2, 1003, 5, B16)
    low["z"][:] = torch.finfo(B16).min
    run_all(low)


def test_infinite_and_missing_values_follow_the_formula():
    s = make(6, 300, 4, F32)
    s["z"][1, 9] = math.nan
    s["z"][2, 9] = math.inf
    s["z"][3] = -math.inf
    s["z"][4, s["index"][4, 1]] = -math.inf  # the teacher wants what the student masks
    loss = mf.train.distill_topk(s["z"], s["teacher"], s["index"])
    assert loss[1].isnan() and loss[2].isnan() and loss[3].isnan() and loss[4] == math.inf
    ok = make(6, 300, 4, F32)
    clean = mf.train.distill_topk(ok["z"], ok["teacher"], ok["index"])
    assert torch.equal(loss[[0, 5]], clean[[0, 5]])
    _, grad = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"])
    assert grad[1:4].isnan().all(1).any() and grad[[0, 4, 5]].isfinite().all()


def test_shapes_strides_and_place():
    s = make(12, 1001, 8, B16)
    want = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"], grad_loss=s["weight"])
    as3 = {n: t.view(3, 4, *t.shape[1:]) for n, t in s.items() if t is not None}
    loss, grad = mf.train.distill_topk_with_grad(as3["z"], as3["teacher"], as3["index"],
                                                 grad_loss=as3["weight"])
    assert loss.shape == (3, 4) and torch.equal(loss.flatten(), want[0])
    assert torch.equal(grad.view(12, 1001), want[1])
    wide = torch.full((12, 1024), 50.0, dtype=B16, device="cuda")
    wide[:, 3:1004] = s["z"]
    cut = wide[:, 3:1004]  # rows apart and off 16-byte boundaries
    loss, grad = mf.train.distill_topk_with_grad(cut, s["teacher"].t().contiguous().t(), s["index"],
                                                 grad_loss=s["weight"])
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[1]) and grad.is_contiguous()
    version = wide._version
    loss, grad = mf.train.distill_topk_with_grad(cut, s["teacher"], s["index"],
                                                 grad_loss=s["weight"], out=cut)
    assert grad is cut and torch.equal(cut, want[1]) and torch.equal(loss, want[0])
    assert wide._version > version
    assert (wide[:, :3] == 50).all() and (wide[:, 1004:] == 50).all()
    columns = s["z"].t().contiguous().t()
    assert torch.equal(mf.train.distill_topk(columns, s["teacher"], s["index"]), want[0])
    number = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"], grad_loss=0.5)[1]
    half = torch.full((12,), 0.5, device="cuda")
    assert torch.equal(number, mf.train.distill_topk_with_grad(
        s["z"], s["teacher"], s["index"], grad_loss=half)[1])
    one = mf.train.distill_topk(s["z"][0], s["teacher"][0], s["index"][0])
    assert one.shape == () and torch.equal(one, want[0][0])


def test_out_that_overlaps_is_refused():
    s = make(4, 100, 3, F32)
    flat = torch.zeros(500, device="cuda")
    z, out = flat[:400].view(4, 100), flat[50:450].view(4, 100)
    with pytest.raises(RuntimeError, match="overlap"):
        mf.train.distill_topk_with_grad(z, s["teacher"], s["index"], out=out)
    with pytest.raises(RuntimeError, match="evenly"):
        mf.train.distill_topk_with_grad(z, s["teacher"], s["index"],
                                        out=torch.zeros(100, 4, device="cuda").t())


def test_empty_and_single_rows():
    z = torch.empty(0, 50, device="cuda", requires_grad=True)
    t, i = torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.int64, device="cuda")
    loss = mf.train.distill_topk(z, t, i)
    loss.sum().backward()
    assert loss.shape == (0,) and z.grad.shape == (0, 50)
    run_all(make(1, 70001, 5, B16))
    run_all(make(700, 300, 2, F32, labels=True), lam=0.1)


def test_same_bits_on_another_stream_and_in_a_graph():
    s = make(40, 5003, 20, B16, labels=True)
    kw = dict(grad_loss=s["weight"], labels=s["labels"], label_weight=0.5)
    want = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"], **kw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"], **kw)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"], **kw)
    for seed in range(3):
        new = make(40, 5003, 20, B16, labels=True, seed=seed + 1)
        for n in s:
            s[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = mf.train.distill_topk_with_grad(s["z"], s["teacher"], s["index"], **kw)
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_gradient_against_differences():
    """Central differences of the weighted loss along a random direction with h = 1/64: the
    loss is smooth with derivatives of order 1 along a direction of unit rms, so truncation
    is about h²; float32 losses of size 10 leave 1e-6 / h: both under 1e-3 of the slope's
    scale |gradient| * |direction| / sqrt(n)."""
    s = make(200, 97, 6, F32, labels=True, seed=4)
    kw = dict(temperature=2.0, labels=s["labels"], label_weight=0.3)

    def total(z):
        loss = mf.train.distill_topk(z, s["teacher"], s["index"], **kw)
        return (loss.double() * s["weight"].double()).sum()

    z = s["z"].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(total(z), z)
    way = g / g.abs().max() + 0.1 * randn(torch.Generator().manual_seed(1), 200, 97).cuda()
    h = 1.0 / 64
    slope = (g.double() * way.double()).sum()
    diff = (total(s["z"] + h * way) - total(s["z"] - h * way)) / (2 * h)
    assert abs(diff - slope) <= 1e-3 * abs(slope)


@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
@pytest.mark.parametrize("v", [777, 20011, 200003])
def test_rows_without_a_term_have_none_of_its_gradient(v, dtype):
    """A term that a row does not have adds nothing to its gradient, whatever its logits are:
    without the first none of softmax(z / tau), without the second none of softmax(z)."""
    s = make(10, v, 6, dtype, labels=True)
    s["labels"][:] = 3
    s["index"][:7] = -1  # no entries
    s["labels"][:4] = -100  # nor a label
    for row, value in enumerate((-math.inf, math.nan, math.inf)):
        s["z"][row, 5 if row else slice(None)] = value
        s["z"][row + 4, 5 if row else slice(None)] = value  # with a label: its term follows the formula
    s["index"][7] = torch.arange(6)  # entries without weight, no label
    s["teacher"][7] = -math.inf
    s["z"][7] = -math.inf
    s["labels"][7:9] = -100  # row 8: only the first term
    loss, grad = run_all(s, tau=1.5, lam=0.4)
    for row in (0, 1, 2, 3, 7):
        assert loss[row] == 0 and not grad[row].any(), row
    for row in (4, 5):
        assert grad[row].isnan().all(), row
    assert grad[8:].isfinite().all()
    bare = dict(s, labels=None)
    _, grad = run_all(bare, tau=1.5)
    for row in range(8):
        assert not grad[row].any(), row


def test_more_rows_than_a_launch_takes():
    """A launch has at most 2^32 - 1 threads, a row up to 1024 of them."""
    rows, v = (1 << 24) + 5, 3
    gen = torch.Generator(device="cuda").manual_seed(0)
    z = torch.randn(rows, v, device="cuda", generator=gen)
    index = torch.randint(0, v, (rows, 1), device="cuda", generator=gen, dtype=torch.int32)
    teacher = torch.zeros(rows, 1, device="cuda")
    labels = torch.randint(-1, v, (rows,), device="cuda", generator=gen)
    weight = torch.rand(rows, device="cuda", generator=gen)
    kw = dict(temperature=2.0, labels=labels, label_weight=0.25)
    want = formula(z, teacher, index, 2.0, labels, 0.25, weight)
    loss, grad = mf.train.distill_topk_with_grad(z, teacher, index, grad_loss=weight, **kw)
    check(loss, want[0], BOUND, "loss")
    check(grad, want[1], BOUND, "gradient")
    z.requires_grad_(True)
    alone = mf.train.distill_topk(z, teacher, index, **kw)
    (auto,) = torch.autograd.grad(alone, z, weight)
    assert torch.equal(alone, loss) and torch.equal(auto, grad)


@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
@pytest.mark.parametrize("v", [300, 20011, 200003])
@pytest.mark.parametrize("labels", [False, True])
def test_rows_whose_softmax_is_nan(v, dtype, labels):
    """A NaN, +inf or -inf everywhere makes the whole of that row's gradient NaN, no other's."""
    s = make(7, v, 4, dtype, labels=True)
    s["labels"][:] = 2
    if not labels:
        s["labels"] = None
    s["z"][1, 9] = math.nan
    s["z"][2, 9] = math.inf
    s["z"][3] = -math.inf
    s["z"][4, s["index"][4, 1]] = -math.inf  # the teacher wants what the student masks
    loss, grad = run_all(s, tau=2.0, lam=0.3)
    assert loss[1:4].isnan().all() and loss[4] == math.inf
    assert grad[1:4].isnan().all() and grad[[0, 4, 5, 6]].isfinite().all()
