"""quantize_fp8, fp8_matmul and fp8_linear on the GPU: the held values and scales bit for bit
against the definition in torch on the CPU, the products against 64 bits, forward and both
gradients, at sizes from one row, column or block to ragged ones past many tiles.

Tolerances: products of held values are exact in float32 up to a sum of K of them, scaled
by s_a * s_b (one rounding each): F32_SUM on the 2-norm, whose terms cancel."""

from __future__ import annotations

import math

import pytest
import torch

import muon_fusion_ascend950_amd as mf
from tests.train_checks import F32_SUM, check, randn

pytestmark = pytest.mark.gpu
F32, B16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def held(x, rows):
    """(values as bytes [R, C padded], scales) by the definition, on the CPU."""
    x = x.detach().float().cpu()
    r, c = x.shape
    rp, cp = -(-r // rows) * rows, -(-c // 128) * 128
    blocks = torch.nn.functional.pad(x, (0, cp - c, 0, rp - r)).view(rp // rows, rows, cp // 128, 128)
    amax = blocks.abs().amax(dim=(1, 3))
    scales = amax * torch.tensor(1 / 448, dtype=F32)
    scales = torch.where(scales < 2.0 ** -126, torch.tensor(2.0 ** -126), scales)
    inverse = torch.ones(()) / scales
    values = (blocks * inverse[:, None, :, None]).to(F8)
    return values.view(rp, cp)[:r].view(torch.uint8), scales


def value(x, rows):
    """What the held matrix stands for, in 64 bits."""
    q, s = held(x, rows)
    s = s.double().repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(128, 1)
    return (q.view(F8).double() * s)[:, : x.shape[1]]


def spread(gen, r, c, dtype=F32):
    """Rows and columns of sizes orders of magnitude apart."""
    return (randn(gen, r, c) * torch.exp(randn(gen, r, 1)) * torch.exp(2 * randn(gen, 1, c))).to(dtype)


@pytest.mark.parametrize("r,c", [(1, 1), (1, 128), (3, 130), (128, 128), (129, 257), (500, 77), (40, 2051)])
@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_bits(r, c, dtype, rows):
    x = spread(torch.Generator().manual_seed(r + c), r, c, dtype)
    got = mf.train.quantize_fp8(x.cuda(), rows)
    values, scales = held(x, rows)
    assert got.shape == (r, c) and got.values.shape == values.shape
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.values.view(torch.uint8).cpu(), values)
    assert torch.equal(got.dequantize().cpu().double(), value(x, rows).float().double())


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_extremes(rows):
    x = torch.zeros(256, 512)
    x[0, 128:256] = 1e-42  # subnormal
    x[128, 0] = 3.4e38
    x[128, 300] = -1e-30
    x[5, 384:] = torch.linspace(-448, 448, 128)  # every rounding of the grid
    x[6, 384:] = torch.linspace(-1, 1, 128) * 2.0 ** -9
    got, (values, scales) = mf.train.quantize_fp8(x.cuda(), rows), held(x, rows)
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.values.view(torch.uint8).cpu() & 0x7f, values & 0x7f)
    x[1, 3] = math.inf
    x[200, 400] = math.nan
    back = mf.train.quantize_fp8(x.cuda(), rows).dequantize().cpu()
    assert back[1, :128].isnan().all() and back[200, 384:].isnan().all()
    ok = torch.ones(256, 512, dtype=torch.bool)
    ok[(slice(0, 128) if rows == 128 else 1), :128] = False
    ok[(slice(128, 256) if rows == 128 else 200), 384:] = False
    assert back[ok].isfinite().all()


def test_quantize_strides():
    gen = torch.Generator().manual_seed(0)
    x = spread(gen, 300, 411)
    for view in (x[7:200:2, 5:301], x.t(), x[:1].expand(40, 411), x[:, :1]):
        g = x.cuda()
        on_gpu = torch.as_strided(g, view.shape, view.stride(), view.storage_offset())
        got, (values, scales) = mf.train.quantize_fp8(on_gpu), held(view, 1)
        assert torch.equal(got.scales.cpu(), scales)
        assert torch.equal(got.values.view(torch.uint8).cpu(), values)


SIZES = [(1, 1, 1), (1, 16, 128), (1, 300, 1000), (2, 5, 129), (16, 64, 256), (17, 130, 640),
         (64, 513, 384), (127, 128, 128), (128, 129, 4096), (150, 2050, 1000), (257, 255, 2050),
         (300, 31, 14336), (1000, 777, 520), (1, 4099, 300), (33, 1, 77), (512, 768, 1024)]


@pytest.mark.parametrize("m,n,k", SIZES, ids=str)
@pytest.mark.parametrize("a_rows,b_rows", [(1, 128), (1, 1), (128, 128)])
def test_products(m, n, k, a_rows, b_rows):
    gen = torch.Generator().manual_seed(m + n + k)
    a, b = spread(gen, m, k), spread(gen, n, k)
    qa, qb = mf.train.quantize_fp8(a.cuda(), a_rows), mf.train.quantize_fp8(b.cuda(), b_rows)
    want = value(a, a_rows) @ value(b, b_rows).t()
    got = mf.train.fp8_matmul(qa, qb, F32)
    assert got.shape == (m, n) and got.dtype == F32
    check(got, want, F32_SUM)
    low = mf.train.fp8_matmul(qa, qb)
    assert low.dtype == B16
    check(low, want, F32_SUM)
    assert torch.equal(got, mf.train.fp8_matmul(qa, qb, F32))


def test_products_of_many_tiles():
    gen = torch.Generator().manual_seed(9)
    a, b = randn(gen, 2100, 900), randn(gen, 1900, 900)
    want = (value(a, 1).cuda() @ value(b, 128).cuda().t())
    qa, qb = mf.train.quantize_fp8(a.cuda()), mf.train.quantize_fp8(b.cuda(), 128)
    check(mf.train.fp8_matmul(qa, qb, F32), want, F32_SUM)
    check(mf.train.fp8_matmul(qb, qa, F32), want.t(), F32_SUM)


def test_exact_sums():
    """Small whole numbers with scales of one: every sum is exact, so every bit is known."""
    gen = torch.Generator().manual_seed(2)
    for m, n, k in ((70, 90, 300), (1, 257, 5000), (300, 520, 1100), (1030, 1290, 640)):
        a = torch.randint(-8, 9, (m, k), generator=gen).float()
        b = torch.randint(-8, 9, (n, k), generator=gen).float()
        qa = mf.train.Fp8Blocks(a.to(F8).cuda(), torch.ones(m, -(-k // 128), device="cuda"))
        qb = mf.train.Fp8Blocks(b.to(F8).cuda(), torch.ones(-(-n // 128), -(-k // 128), device="cuda"))
        assert torch.equal(mf.train.fp8_matmul(qa, qb, F32).cpu(), a @ b.t())


@pytest.mark.parametrize("m,n,k", [(4100, 4610, 256), (4360, 4501, 640), (4608, 4608, 384), (2200, 2300, 200)])
def test_workgroups_of_several_tiles(m, n, k):
    """bf16 results of more tiles than compute units.  Ones and zeros of both signs: a block's
    sums are whole numbers up to 128, far above what the fp8 MFMAs lose, the total is exact in
    fp32 and rounded once."""
    gen = torch.Generator().manual_seed(k)
    a = torch.randint(-1, 2, (m, k), generator=gen).float().cuda()
    b = torch.randint(-1, 2, (n, k), generator=gen).float().cuda()
    blocks = -(-k // 128)
    qa = mf.train.Fp8Blocks(a.to(F8), torch.ones(m, blocks, device="cuda"))
    qb = mf.train.Fp8Blocks(b.to(F8), torch.ones(-(-n // 128), blocks, device="cuda"))
    want = (a @ b.t()).to(B16)
    for _ in range(3):
        assert torch.equal(mf.train.fp8_matmul(qa, qb, B16), want)


@pytest.mark.parametrize("m,n,k", [(17, 64, 2700), (32, 1000, 5000), (64, 4096, 4096), (65, 129, 128 * 23),
                                   (100, 1, 4000), (130, 2050, 2560)])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
def test_split_products(m, n, k, b_rows, dtype):
    """Few tiles of a long K: the parts of K meet in the parts' order."""
    gen = torch.Generator().manual_seed(m + n + k)
    a, b = spread(gen, m, k, F32), randn(gen, n, k)
    want = value(a, 1).cuda() @ value(b, b_rows).cuda().t()
    qa, qb = mf.train.quantize_fp8(a.cuda()), mf.train.quantize_fp8(b.cuda(), b_rows)
    got = mf.train.fp8_matmul(qa, qb, dtype)
    check(got, want, F32_SUM)
    assert torch.equal(got, mf.train.fp8_matmul(qa, qb, dtype))


def test_split_product_of_a_nan_row_and_in_a_graph():
    gen = torch.Generator().manual_seed(8)
    a, b = randn(gen, 40, 5000), randn(gen, 300, 5000)
    qb = mf.train.quantize_fp8(b.cuda(), 128)
    clean = mf.train.fp8_matmul(mf.train.quantize_fp8(a.cuda()), qb)
    a[7, 4990] = math.nan
    x = a.cuda()
    qa = mf.train.quantize_fp8(x)
    got = mf.train.fp8_matmul(qa, qb)
    rows = [i for i in range(40) if i != 7]
    assert got[7].isnan().all() and torch.equal(got[rows], clean[rows])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mf.train.fp8_matmul(mf.train.quantize_fp8(x), qb)
    for step in range(4):
        x.copy_(randn(gen, 40, 5000))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, mf.train.fp8_matmul(mf.train.quantize_fp8(x), qb)), step


def test_each_block_has_its_scale():
    """One element of a in each block of 128, scales that are powers of two of their place:
    the product of one block with ones, exactly."""
    m, n, k = 200, 300, 5 * 128
    for b_rows in (1, 128):
        sa = 2.0 ** ((torch.arange(m)[:, None] * 3 + torch.arange(5)) % 11 - 5).float()
        nb = n if b_rows == 1 else -(-n // 128)
        sb = 2.0 ** ((torch.arange(nb)[:, None] * 5 + 2 * torch.arange(5)) % 7 - 3).float()
        a = torch.zeros(m, k)
        for block in range(5):
            a[:, block * 128 + (torch.arange(m).argmax() * 0 + 31 * block) % 128] = 1.0 + block
        b = torch.ones(n, k)
        qa = mf.train.Fp8Blocks(a.to(F8).cuda(), sa.cuda())
        qb = mf.train.Fp8Blocks(b.to(F8).cuda(), sb.cuda())
        full = sb.repeat_interleave(b_rows, 0)[:n]
        want = (sa * torch.arange(1.0, 6.0)) @ full.t()
        assert torch.equal(mf.train.fp8_matmul(qa, qb, F32).cpu(), want)


def test_rows_of_nan_and_padding():
    """A NaN stays in its row; bytes past a matrix's own columns are no part of it."""
    gen = torch.Generator().manual_seed(3)
    a, b = randn(gen, 40, 300), randn(gen, 70, 300)
    clean = mf.train.fp8_matmul(mf.train.quantize_fp8(a.cuda()), mf.train.quantize_fp8(b.cuda(), 128))
    a[11, 200] = math.nan
    got = mf.train.fp8_matmul(mf.train.quantize_fp8(a.cuda()), mf.train.quantize_fp8(b.cuda(), 128))
    rows = [i for i in range(40) if i != 11]
    assert got[11].isnan().all() and torch.equal(got[rows], clean[rows])
    wide = torch.full((70, 384), 0x7f, dtype=torch.uint8, device="cuda")  # NaN past column 300
    qb = mf.train.quantize_fp8(b.cuda(), 128)
    wide[:, :300] = qb.values.view(torch.uint8)[:, :300]
    cut = mf.train.Fp8Blocks(wide[:, :300].view(F8), qb.scales)
    got = mf.train.fp8_matmul(mf.train.quantize_fp8(a.cuda()), cut)
    assert torch.equal(got[rows], clean[rows])


def test_operands_of_other_layouts():
    gen = torch.Generator().manual_seed(4)
    a, b = mf.train.quantize_fp8(randn(gen, 50, 500).cuda()), mf.train.quantize_fp8(randn(gen, 300, 500).cuda(), 128)
    want = mf.train.fp8_matmul(a, b)
    rows = mf.train.Fp8Blocks(a.values, a.scales.contiguous(), a.shape)
    wide = torch.zeros(50, 527, dtype=torch.uint8, device="cuda")
    wide[:, 3:515] = a.values.view(torch.uint8)
    shifted = mf.train.Fp8Blocks(wide[:, 3:515].view(F8), a.scales, a.shape)
    turned = mf.train.Fp8Blocks(b.values, b.scales.t().contiguous().t(), b.shape)
    for x, y in ((rows, b), (shifted, b), (a, turned)):
        assert torch.equal(mf.train.fp8_matmul(x, y), want)


LINEAR = [((1,), 128, 128), ((1, 1), 300, 260), ((3, 50), 130, 1000), ((5, 7), 513, 77),
          ((333,), 768, 2050), ((2, 260), 640, 384), ((1200,), 520, 650)]


@pytest.mark.parametrize("lead,n,k", LINEAR, ids=str)
@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (B16, F32), (B16, B16)], ids=str)
def test_linear_and_gradients(lead, n, k, dtype, weight_dtype):
    gen = torch.Generator().manual_seed(n + k)
    t = math.prod(lead)
    x, w = spread(gen, t, k, dtype), (randn(gen, n, k) / math.sqrt(k)).to(weight_dtype)
    dy = spread(gen, t, n, dtype)
    xg = x.view(*lead, k).cuda().requires_grad_(True)
    wg = w.cuda().requires_grad_(True)
    y = mf.train.fp8_linear(xg, wg)
    assert y.shape == (*lead, n) and y.dtype == dtype
    check(y.view(t, n), value(x, 1) @ value(w, 128).t(), F32_SUM, "y")
    with torch.no_grad():
        assert torch.equal(mf.train.fp8_linear(xg, wg), y)
        assert torch.equal(mf.train.fp8_linear(xg, mf.train.quantize_fp8(wg, 128)), y)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.view(*lead, n).cuda())
    assert dx.shape == xg.shape and dx.dtype == dtype and dw.shape == w.shape and dw.dtype == weight_dtype
    check(dx.view(t, k), value(dy, 1) @ value(w, 128), F32_SUM, "dx")
    check(dw, value(dy.t(), 1) @ value(x.t(), 1).t(), F32_SUM, "dw")


def test_only_some_gradients_wanted():
    gen = torch.Generator().manual_seed(6)
    x, w, dy = spread(gen, 70, 300).cuda(), randn(gen, 140, 300).cuda(), randn(gen, 70, 140).cuda()
    both = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(mf.train.fp8_linear(*both), both, dy)
    a = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(mf.train.fp8_linear(a, w), a, dy)[0], dx)
    b = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(mf.train.fp8_linear(x, b), b, dy.t().contiguous().t())[0], dw)


def test_no_tokens():
    x = torch.empty(0, 3, 256, device="cuda", requires_grad=True)
    w = torch.randn(100, 256, device="cuda", requires_grad=True)
    y = mf.train.fp8_linear(x, w)
    y.sum().backward()
    assert y.shape == (0, 3, 100) and x.grad.shape == x.shape
    assert torch.equal(w.grad, torch.zeros_like(w))


def test_gradients_against_differences():
    """The product is linear in each operand but for its rounding to 8 bits, 2^-4 of a value
    at most: along the gradient itself the change over a step of the operand's own size is
    the slope to within that."""
    gen = torch.Generator().manual_seed(8)
    x, w = randn(gen, 200, 384).cuda(), randn(gen, 256, 384).cuda()
    dy = randn(gen, 200, 256).cuda()
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(mf.train.fp8_linear(xg, wg), (xg, wg), dy)

    def total(a, b):
        with torch.no_grad():
            return (mf.train.fp8_linear(a, b).double() * dy.double()).sum()

    for g, at in ((dx, lambda d: total(x + d, w)), (dw, lambda d: total(x, w + d))):
        way = g / g.square().mean().sqrt()
        slope = (g.double() * way.double()).sum()
        assert abs((at(way) - at(-way)) / 2 - slope) <= 2.0 ** -4 * slope


def test_another_stream_and_a_graph():
    gen = torch.Generator().manual_seed(7)
    x, w = randn(gen, 200, 640, dtype=B16).cuda(), mf.train.quantize_fp8(randn(gen, 512, 640).cuda(), 128)
    want = mf.train.fp8_linear(x, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = mf.train.fp8_linear(x, w)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    for rows in (1, 200):
        held_x = x[:rows].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mf.train.fp8_linear(held_x, w)
        for _ in range(3):
            held_x.copy_(randn(gen, rows, 640, dtype=B16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, mf.train.fp8_linear(held_x, w))


@pytest.mark.parametrize("m", [1, 2, 3, 15, 16, 17])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 100), (16, 128), (100, 1024), (129, 1100), (8210, 700),
                                 (300, 14336)])
@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
def test_few_tokens(m, n, k, dtype):
    """Up to 16 tokens are quantised in the product's own kernel: the bits of the two calls,
    and each token's result is its own whatever the others are."""
    gen = torch.Generator().manual_seed(m + n + k)
    x, w = spread(gen, m, k, dtype), randn(gen, n, k)
    q = mf.train.quantize_fp8(w.cuda(), 128)
    got = mf.train.fp8_linear(x.cuda(), q)
    check(got, value(x, 1) @ value(w, 128).t(), F32_SUM)
    two = mf.train.fp8_matmul(mf.train.quantize_fp8(x.cuda()), q, dtype)
    assert torch.equal(got, two)
    x[1:] *= math.inf
    assert torch.equal(mf.train.fp8_linear(x.cuda(), q)[0], got[0])
    wide = torch.full((m, k + 3), 7.0, dtype=dtype, device="cuda")
    wide[:, 3:] = x.cuda()
    assert torch.equal(mf.train.fp8_linear(wide[:, 3:], q)[0], got[0])


@pytest.mark.parametrize("m,n,k", [(1, 300, 9000), (4, 40, 12288), (12, 8200, 4096), (13, 100, 4000), (5, 70, 4097)])
@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
def test_few_tokens_of_long_rows(m, n, k, dtype):
    """Both sides of the sizes up to which the product's own kernel quantises."""
    gen = torch.Generator().manual_seed(m + n + k)
    x, w = spread(gen, m, k, dtype), randn(gen, n, k)
    q = mf.train.quantize_fp8(w.cuda(), 128)
    got = mf.train.fp8_linear(x.cuda(), q)
    check(got, value(x, 1) @ value(w, 128).t(), F32_SUM)
    assert torch.equal(got, mf.train.fp8_matmul(mf.train.quantize_fp8(x.cuda()), q, dtype))


def kernel_names(f):
    """Names of the kernels that `f` launches, from a graph of them."""
    import ctypes

    class Params(ctypes.Structure):
        _fields_ = [("block", ctypes.c_uint32 * 3), ("extra", ctypes.c_void_p), ("func", ctypes.c_void_p),
                    ("grid", ctypes.c_uint32 * 3), ("params", ctypes.c_void_p), ("shared", ctypes.c_uint32)]

    f()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        f()
    with open("/proc/self/maps") as maps:
        hip = ctypes.CDLL(next(line.split()[-1] for line in maps if "libamdhip64.so" in line))
    hip.hipKernelNameRefByPtr.restype = ctypes.c_char_p
    handle, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(handle, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert hip.hipGraphGetNodes(handle, nodes, ctypes.byref(count)) == 0
    names = []
    for node in nodes:
        p = Params()
        assert hip.hipGraphKernelNodeGetParams(ctypes.c_void_p(node), ctypes.byref(p)) == 0
        names.append(hip.hipKernelNameRefByPtr(ctypes.c_void_p(p.func), None).decode())
    return names


TILED = [(2000, 4000, 640, 128), (4100, 4610, 256, 128), (4500, 4700, 512, 256), (4608, 4608, 256, 256)]
TILED_F32 = [(2000, 4000, 640, 128), (4000, 4090, 384, 256), (4096, 4096, 256, 256)]


@pytest.mark.parametrize("m,n,k,side,dtype", [(*s, B16) for s in TILED] + [(*s, F32) for s in TILED_F32], ids=str)
@pytest.mark.parametrize("b_rows", [1, 128])
def test_scales_of_large_tiles(m, n, k, side, dtype, b_rows):
    """Ones and zeros of both signs, scales that are powers of two drawn for each row, column
    block and block of K: whole and ragged tiles, several a workgroup, two steps and more.  Every
    sum is a multiple of 2^-4 below 2^15: exact in fp32, rounded once to bf16."""
    gen = torch.Generator().manual_seed(m + k + b_rows)
    blocks, nb = -(-k // 128), n if b_rows == 1 else -(-n // 128)
    a = torch.randint(-1, 2, (m, k), generator=gen).float()
    b = torch.randint(-1, 2, (n, k), generator=gen).float()
    sa = torch.exp2(torch.randint(-2, 3, (m, blocks), generator=gen).float())
    sb = torch.exp2(torch.randint(-2, 3, (nb, blocks), generator=gen).float())
    qa = mf.train.Fp8Blocks(a.to(F8).cuda(), sa.cuda())
    qb = mf.train.Fp8Blocks(b.to(F8).cuda(), sb.cuda())
    want = (qa.dequantize().double() @ qb.dequantize().double().t()).to(dtype)
    names = kernel_names(lambda: mf.train.fp8_matmul(qa, qb, dtype))
    assert any(f"matmul_kernelILi{side}ELi{side}E" in name for name in names), names
    for _ in range(2):
        assert torch.equal(mf.train.fp8_matmul(qa, qb, dtype), want)


# few rows, 64 x 64 tiles, those split along K, 128 x 128 and 256 x 256
FAR = [(3, 70, 384), (70, 90, 384), (32, 300, 5120), (2000, 4000, 384)]


def far_scales(kind, m, n, k, b_rows, gen):
    """Values and scales whose products s_a * s_b leave float32 where the results do not."""
    blocks, nb = k // 128, n if b_rows == 1 else -(-n // 128)

    def scales(rows, exponents):
        e = torch.tensor([exponents[i % len(exponents)] for i in range(blocks)])
        return (1 + torch.rand(rows, blocks, generator=gen)) * torch.exp2(e.float())

    a = torch.randint(0, 2, (m, k), generator=gen).float()
    b = torch.randint(0, 2, (n, k), generator=gen).float()
    if kind == "small":  # s_a * s_b about 2^-144, results from 2^-122 on
        return 256 * a, 256 * b, scales(m, [-72]), scales(nb, [-73])
    if kind == "large":  # s_a * s_b about 2^131, results about 2^125
        return a * 2.0 ** -9, b * 2.0 ** -6, scales(m, [119]), scales(nb, [11])
    # blocks of zero sums with s_a * s_b about 2^202, beside others
    a[:, ::2] = torch.where((torch.arange(0, k, 2) // 128 % 2 == 0), 0.0, a[:, ::2])
    b[:, 1::2] = torch.where((torch.arange(1, k, 2) // 128 % 2 == 0), 0.0, b[:, 1::2])
    return a, b, scales(m, [101, 70]), scales(nb, [100, -72])


@pytest.mark.parametrize("kind", ["small", "large", "zero"])
@pytest.mark.parametrize("m,n,k,dtype", [(*s, d) for s in FAR for d in (F32, B16)] +
                         [(4000, 4090, 384, F32), (4500, 4700, 384, B16)], ids=str)
@pytest.mark.parametrize("b_rows", [1, 128])
def test_scales_far_apart(kind, m, n, k, dtype, b_rows):
    """Products of two scales under and over float32's range, of results inside it.  A block's
    sum has one rounding, its scales two, the sum of blocks one each: the bounds above."""
    gen = torch.Generator().manual_seed(m + n + k)
    a, b, sa, sb = far_scales(kind, m, n, k, b_rows, gen)
    qa = mf.train.Fp8Blocks(a.to(F8).cuda(), sa.cuda())
    qb = mf.train.Fp8Blocks(b.to(F8).cuda(), sb.cuda())

    def exact(q, values, rows):
        s = q.scales.double().repeat_interleave(rows, 0)[: values.shape[0]]
        return values.cuda().double() * s.repeat_interleave(128, 1)

    want = exact(qa, a, 1) @ exact(qb, b, b_rows).t()
    assert torch.isfinite(want.to(dtype)).all()
    check(mf.train.fp8_matmul(qa, qb, dtype), want, F32_SUM, kind)


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("dtype", [F32, B16], ids=str)
def test_linear_of_values_far_apart(rows, dtype):
    """Large values that meet zeros, and the smallest beside them, forward and both gradients."""
    gen = torch.Generator().manual_seed(rows)
    x, w, dy = randn(gen, rows, 384, dtype=dtype), randn(gen, 200, 384), randn(gen, rows, 200, dtype=dtype)
    x[:, :128], w[:, :128] = 0.0, 0.0
    x[:, 0], w[:, 1] = 2.0 ** 120, 2.0 ** 40
    x[:, 256:], w[:, 256:] = x[:, 256:] * 2.0 ** -70, w[:, 256:] * 2.0 ** -72
    dy[:, 128:] = 0.0
    dy[0], dy[1:, 0] = 0.0, 2.0 ** 40  # the weight's gradient sums over rows
    x[1:, 0] = 0.0
    check(mf.train.fp8_linear(x.cuda(), mf.train.quantize_fp8(w.cuda(), 128)),
          value(x, 1) @ value(w, 128).t(), F32_SUM, "held")
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = mf.train.fp8_linear(xg, wg)
    check(y, value(x, 1) @ value(w, 128).t(), F32_SUM, "y")
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.cuda())
    check(dx, value(dy, 1) @ value(w, 128), F32_SUM, "dx")
    check(dw, value(dy.t(), 1) @ value(x.t(), 1).t(), F32_SUM, "dw")


@pytest.mark.parametrize("m,n,k", [(3, 70, 1000), (70, 90, 1000), (32, 300, 5000), (2000, 4000, 400), (4500, 4700, 400)],
                         ids=str)
@pytest.mark.parametrize("b_rows", [1, 128])
def test_what_bf16_results_keep_of_a_sum(m, n, k, b_rows):
    """Element by element, with outliers among the values: eight products at a time are cut off
    below 2^-13 of their largest, so a sum is off by at most 7 * 2^-13 of the sum of magnitudes,
    and the sum of blocks in fp32 by 2^-20 of it; the result is the rounding of such a sum."""
    gen = torch.Generator().manual_seed(m + k)
    a, b = randn(gen, m, k), randn(gen, n, k)
    a[:, ::11], b[:, ::13] = a[:, ::11] * 100, b[:, ::13] * 30
    qa, qb = mf.train.quantize_fp8(a.cuda()), mf.train.quantize_fp8(b.cuda(), b_rows)
    va, vb = value(a, 1).cuda(), value(b, b_rows).cuda()
    exact, size = va @ vb.t(), va.abs() @ vb.abs().t()
    off = (7 * 2.0 ** -13 + 2.0 ** -20) * size
    got = mf.train.fp8_matmul(qa, qb)
    assert (got >= (exact - off).to(B16)).all() and (got <= (exact + off).to(B16)).all()
    off = (mf.train.fp8_matmul(qa, qb, F32).double() - exact).abs()
    assert (off <= 2.0 ** -18 * size).all()  # at most 80 sums and roundings of 2^-24 behind another
