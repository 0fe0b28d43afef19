"""GPU parity of 4-bit matrices (tri_fp4_quantize, tri_fp4_dequantize) and of products over them (tri_fp4_matmul) with
oracle/experts.py, which computes in fp64.  Codes and values are compared exactly, products within the bound of their roundings
(experts_util.product_tolerance).  What lies between the rows of scales holds 255, which reads as NaN."""
import math

import pytest
import torch

from cache_util import assert_within
from experts_util import four_bit, lay_scales, product_tolerance, to_dev
from oracle import cache as oc
from oracle import experts as oe
from trinity_amd import blocks, ext

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _x(g, M, K, dtype, pad=0):
    x = torch.randn(M, K + pad, generator=g) * torch.exp(0.5 * torch.randn(K + pad, generator=g))
    return x.to(dtype)[:, :K]


@pytest.mark.parametrize("M,K,pad", [(1, 32, 0), (3, 96, 8), (17, 4544, 0), (70000, 32, 0), (130, 18176, 16), (300, 7232, 0)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantize_and_back(dev, M, K, pad, dtype):
    g = torch.Generator().manual_seed(M + K)
    x = _x(g, M, K, dtype, pad)
    if M > 2:
        x[1, :32] = 0
        x[2, 3], x[2, K - 1] = math.inf, math.nan
        x[0, 0] = torch.finfo(dtype).max
        x[0, 33:40] = torch.finfo(dtype).smallest_normal / 8
    codes, scales = blocks.Fp4Matmul.quantize(to_dev(x, dev))
    want = oc.fp4_encode(x)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    values = oc.fp4_decode(*want)
    for t in (F16, BF16):
        got = blocks.Fp4Matmul.dequantize(codes, scales, t)
        assert got.dtype == t and torch.equal(got.cpu().isnan(), values.isnan())
        assert torch.equal(got.cpu().nan_to_num(0, 9, -9), values.to(t).nan_to_num(0, 9, -9))


def test_quantize_into_strided_rows(dev):
    """Rows of codes and scales that are parts of larger buffers: what is between them stays."""
    g = torch.Generator().manual_seed(5)
    x = _x(g, 37, 160, F16)
    want = oc.fp4_encode(x)
    codes, scales = torch.full((37, 96), 7, dtype=torch.uint8), torch.full((37 * 9 + 3,), 7, dtype=torch.uint8)
    dc, ds = codes.to(dev), scales.to(dev)
    ext.fp4_quantize(x.to(dev), dc[:, :80], ds[3:].view(37, 9)[:, :5])
    codes[:, :80], scales[3:].view(37, 9)[:, :5] = want
    assert torch.equal(dc.cpu(), codes) and torch.equal(ds.cpu(), scales)
    y = torch.full((37, 200), 5, dtype=BF16, device=dev)
    ext.fp4_dequantize(dc[:, :80], ds[3:].view(37, 9)[:, :5], y[:, 8:168])
    assert torch.equal(y[:, 8:168].cpu().double(), oc.fp4_decode(*want))
    assert bool((y[:, :8] == 5).all()) and bool((y[:, 168:] == 5).all())


# M, K, N; scales: bytes between rows, and of the first row from an aligned address
PRODUCTS = [
    (1, 32, 8, 0, 0), (1, 256, 24, 0, 0), (1, 4096, 136, 3, 5), (2, 288, 40, 0, 1), (16, 1120, 200, 1, 0), (5, 2272, 24, 0, 0),
    (16, 224, 8, 0, 0), (17, 256, 264, 0, 0), (17, 32, 8, 0, 0), (32, 4544, 520, 0, 0), (33, 96, 120, 2, 3), (64, 544, 136, 0, 7),
    (65, 1824, 264, 0, 0), (128, 2048, 128, 0, 0), (129, 64, 264, 5, 1), (200, 800, 1000, 0, 0), (256, 320, 512, 0, 0),
    (257, 1056, 264, 0, 0), (300, 4544, 520, 0, 0), (513, 288, 776, 1, 2), (700, 96, 3000, 0, 0), (1030, 544, 1032, 0, 0),
]


@pytest.mark.parametrize("M,K,N,pad,shift", PRODUCTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("x4", [False, True])
def test_product(dev, M, K, N, pad, shift, dtype, x4):
    g = torch.Generator().manual_seed(M * 7 + K + N)
    w, ws = four_bit(g, N, K, std=0.05, pad=pad, shift=shift)
    x = _x(g, M, K, dtype, 8)
    dw, dws = to_dev(w, dev), to_dev(ws, dev)
    if x4:
        codes, scales = oc.fp4_encode(x)
        want, mag = oe.fp4_matmul(codes, w, ws, scales)
        got = blocks.Fp4Matmul().run(codes.to(dev), dw, dws, x_scales=to_dev(lay_scales(scales, pad, shift), dev), dtype=dtype)
        again = blocks.Fp4Matmul(quantize_x=True).run(to_dev(x, dev), dw, dws)
        assert torch.equal(got, again)
    else:
        want, mag = oe.fp4_matmul(x, w, ws)
        got = blocks.Fp4Matmul().run(to_dev(x, dev), dw, dws)
    assert got.dtype == dtype
    tol = product_tolerance(want, mag, K, dtype)
    assert_within(got, want, tol, "product")
    # without room for parts of K, into rows of a larger buffer
    big = torch.full((M, N + 16), 3, dtype=dtype, device=dev)
    a = (codes.to(dev), scales.to(dev)) if x4 else (to_dev(x, dev), None)
    ext.fp4_matmul(*a, dw, dws, None, big[:, 8:N + 8])
    assert_within(big[:, 8:N + 8], want, tol, "product without a workspace")
    assert bool((big[:, :8] == 3).all()) and bool((big[:, N + 8:] == 3).all())


# M, K, N, x in 4 bits: a product for each tile, number of row blocks in it, and whole K or parts (test_experts_plans.py)
FORMS = [
    (200, 96, 8200, True), (20, 8224, 4104, True), (20, 96, 136, True), (33, 2080, 136, True), (1000, 96, 2056, True),
    (70, 4128, 4104, True), (1000, 96, 8200, True), (333, 14336, 8192, True),
    (20, 96, 136, False), (20, 2080, 136, False), (400, 96, 8200, False), (257, 8224, 4104, False), (1000, 96, 2056, False),
    (2500, 4128, 264, False), (1300, 96, 8200, False), (40, 4128, 8200, False), (70, 8224, 8200, False), (130, 8224, 8200, False),
    (1000, 96, 8200, False), (1, 96, 136, False), (1, 544, 136, False), (4, 4544, 136, False), (3, 36896, 72, False),
    (16, 800, 200, False), (16, 18176, 136, False), (1, 90016, 40, False),
]


@pytest.mark.parametrize("M,K,N,x4", FORMS)
def test_product_in_every_form(dev, M, K, N, x4):
    g = torch.Generator().manual_seed(M + K + N)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    ws = torch.randint(117, 124, (N, K // 32), generator=g, dtype=torch.uint8)
    x, op = _x(g, M, K, BF16), blocks.Fp4Matmul(quantize_x=x4)
    rows, xs = oc.fp4_encode(x) if x4 else (x, None)
    want, mag = oe.fp4_matmul(rows, w, ws, xs)
    got = op.run(x.to(dev), w.to(dev), ws.to(dev))
    assert_within(got, want, product_tolerance(want, mag, K, BF16), "product")


@pytest.mark.parametrize("M,K", [(1, 81600), (1, 81664), (1, 90016), (3, 90016), (16, 90016), (16, 18176), (17, 90016)])
def test_long_rows_without_a_workspace(dev, M, K):
    """Rows of which the LDS holds none, or one as a whole."""
    N, g = 40, torch.Generator().manual_seed(K)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    ws = torch.randint(117, 124, (N, K // 32), generator=g, dtype=torch.uint8)
    x, out = _x(g, M, K, BF16), torch.zeros(M, N, dtype=BF16, device=dev)
    want, mag = oe.fp4_matmul(x, w, ws)
    for room in (None, torch.empty(256, dtype=torch.uint8, device=dev)):
        ext.fp4_matmul(x.to(dev), None, w.to(dev), ws.to(dev), room, out)
        assert_within(out, want, product_tolerance(want, mag, K, BF16), "product")


@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("x4", [False, True])
def test_every_value_of_k_counts_once(dev, M, x4):
    """x is one at one value of K and zero elsewhere: out is that column of the weights, exactly."""
    K, N = 1120, 72
    g = torch.Generator().manual_seed(M)
    w, ws = four_bit(g, N, K)
    values = oc.fp4_decode(w, ws)
    at = [0, 1, 31, 32, 63, 64, 127, 255, 256, 511, 512, 1023, 1024, 1087, 1088, 1119] + list(range(5, K, 53))
    op, dw, dws = blocks.Fp4Matmul(quantize_x=x4), w.to(dev), ws.to(dev)
    for i in range(0, len(at), M):
        x = torch.zeros(M, K, dtype=F16)
        for r, k in enumerate(at[i:i + M]):
            x[r, k] = 1
        got = op.run(x.to(dev), dw, dws).cpu().double()
        for r, k in enumerate(at[i:i + M]):
            assert torch.equal(got[r], values[:, k].half().double()), k
        assert bool((got[len(at[i:i + M]):] == 0).all())


@pytest.mark.parametrize("M", [3, 20, 300])
@pytest.mark.parametrize("x4", [False, True])
def test_values_that_are_no_numbers_stay_in_their_row_and_column(dev, M, x4):
    K, N = 352, 136
    g = torch.Generator().manual_seed(9)
    w, ws = four_bit(g, N, K)
    x = _x(g, M, K, BF16)
    x[1, 7], x[2, K - 1] = math.nan, math.inf
    ws[5, 3], ws[N - 1, K // 32 - 1] = 255, 255
    got = blocks.Fp4Matmul(quantize_x=x4).run(x.to(dev), w.to(dev), ws.to(dev)).cpu()
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[1:3], bad[:, 5], bad[:, N - 1] = True, True, True
    assert torch.equal(~torch.isfinite(got), bad)
    if not x4:
        zero = oc.fp4_decode(w, ws)[:, K - 1] == 0
        keep = ~zero
        keep[5] = keep[N - 1] = False
        assert bool(torch.isinf(got[2][keep]).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_code_at_every_scale(dev, dtype):
    """What the element type cannot hold counts as the type has it: subnormals, zeros, infinities; 255 is NaN."""
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(1, 256).repeat(256, 1)      # both halves of a byte
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(256, 1).repeat(1, 16)
    want = oc.fp4_decode(codes, scales).to(dtype)
    got = blocks.Fp4Matmul.dequantize(codes.to(dev), scales.to(dev), dtype).cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 16, 40, 300])
@pytest.mark.parametrize("x4", [False, True])
def test_products_at_every_scale(dev, dtype, M, x4):
    """One value of K at a time against weights of every scale whose values the type holds as normal numbers."""
    lo, hi = (127 - 13, 127 + 13) if dtype == F16 else (127 - 100, 127 + 100)
    N, K = hi - lo + 1 + (-(hi - lo + 1)) % 8, 512
    g = torch.Generator().manual_seed(M)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (lo + torch.arange(N) % (hi - lo + 1)).to(torch.uint8).view(N, 1).repeat(1, K // 32)
    x = torch.zeros(M, K, dtype=dtype)
    at = torch.randint(0, K, (M,), generator=g)
    x[torch.arange(M), at] = 1
    got = blocks.Fp4Matmul(quantize_x=x4).run(x.to(dev), codes.to(dev), scales.to(dev)).cpu()
    assert torch.equal(got, oc.fp4_decode(codes, scales)[:, at].t().to(dtype))


def test_empty(dev):
    w, ws = four_bit(torch.Generator().manual_seed(1), 16, 64)
    op = blocks.Fp4Matmul()
    assert op.run(torch.empty(0, 64, dtype=F16, device=dev), w.to(dev), ws.to(dev)).shape == (0, 16)
    codes, scales = op.quantize(torch.empty(0, 64, dtype=BF16, device=dev))
    assert codes.shape == (0, 32) and scales.shape == (0, 2)
    assert op.dequantize(codes, scales).shape == (0, 64)


@pytest.mark.parametrize("M", [1, 100])
@pytest.mark.parametrize("x4", [False, True])
def test_captured_and_replayed(dev, M, x4):
    K, N = 2048, 256
    g = torch.Generator().manual_seed(3)
    w, ws = four_bit(g, N, K)
    dw, dws, x = w.to(dev), ws.to(dev), torch.zeros(M, K, dtype=F16, device=dev)
    op = blocks.Fp4Matmul(quantize_x=x4)
    op.run(x, dw, dws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op.run(x, dw, dws)
    for i in range(4):
        new = _x(torch.Generator().manual_seed(i), M, K, F16).to(dev)
        x.copy_(new)
        graph.replay()
        eager = op.run(new, dw, dws)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_on_another_stream(dev):
    g = torch.Generator().manual_seed(4)
    w, ws = four_bit(g, 512, 4096)
    x = _x(g, 40, 4096, BF16).to(dev)
    dw, dws = w.to(dev), ws.to(dev)
    op = blocks.Fp4Matmul()
    want = op.run(x, dw, dws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [op.run(x, dw, dws) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for y in got)
