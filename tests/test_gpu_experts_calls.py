"""GPU: calls of blocks.Router, Fp4Matmul and ExpertsFfn at the borders of what they take, against oracle/experts.py."""
import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from cache_util import UNIT, assert_within
from experts_util import sums, to_dev
from oracle import cache as oc
from oracle import experts as oe
from test_gpu_experts import _ids, _weights
from trinity_amd import blocks, ext

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (1, 1, 1), (70, 16, 4), (33, 128, 8), (40, 256, 8)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_what_a_group_counts_means_nothing_where_there_is_one(dev, T, E, k, scores):
    g = torch.Generator().manual_seed(T + E)
    z, b = 1.5 * torch.randn(T, E, generator=g), 0.3 * torch.randn(E, generator=g)
    ids, weights = blocks.Router(k, scores=scores, group_top=2, scale=2.5).route(z.to(dev), b.to(dev))
    want, w = oe.route(z, b, top_k=k, sigmoid=scores == "sigmoid", scale=2.5)
    assert torch.equal(ids.cpu().long(), want)
    assert_within(weights, w, 2.0 ** -24 * w.abs() * 1.01, "weights")


@pytest.mark.parametrize("E,groups,top_groups", [(7, 1, 1), (12, 1, 1), (12, 3, 2), (30, 1, 1), (64, 1, 1), (64, 8, 1), (100, 1, 1),
                                                 (256, 8, 2), (400, 1, 1)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_a_nan_makes_its_tokens_weights_nan(dev, E, groups, top_groups, sigmoid, renormalize):
    """Of whichever expert it is - chosen, passed over or in a group that goes - and no other token's."""
    g, k = torch.Generator().manual_seed(E), 3
    z = torch.randn(45, E, generator=g)
    bad = torch.arange(45) % 4 == 1
    for i, t in enumerate(bad.nonzero().flatten().tolist()):
        z[t, (0, E - 1, E // 2, int(z[t].argmin()), int(z[t].argmax()))[i % 5]] = math.nan
    op = blocks.Router(k, scores="sigmoid" if sigmoid else "softmax", groups=groups, top_groups=top_groups, renormalize=renormalize)
    ids, w = (t.cpu() for t in op.route(z.to(dev)))
    assert torch.equal(w.isnan(), bad[:, None].expand(45, k))
    assert bool((ids.sort(-1).values.diff(dim=-1) > 0).all()) and bool(((ids >= 0) & (ids < E)).all())
    want, value = oe.route(z[~bad], top_k=k, sigmoid=sigmoid, groups=groups, top_groups=top_groups, renormalize=renormalize)
    assert torch.equal(ids[~bad].long(), want)
    assert_within(w[~bad], value, 2.0 ** -24 * value * 1.01, "weights")
    bias = torch.zeros(E)
    bias[E // 3] = math.nan  # (every token's)
    ids, w = (t.cpu() for t in op.route(z.to(dev), bias.to(dev)))
    assert bool(w.isnan().all())
    assert bool((ids.sort(-1).values.diff(dim=-1) > 0).all()) and bool(((ids >= 0) & (ids < E)).all())


@pytest.mark.parametrize("T,E,k,N,F,how", [(416, 2, 1, 96, 160, "spread"), (512, 2, 1, 96, 160, "spread"), (514, 2, 1, 96, 160, "spread"),
                                           (384, 1, 1, 64, 544, "spread"), (385, 1, 1, 64, 544, "spread"), (770, 6, 3, 64, 96, "one")])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_four_bit_experts_where_their_tiles_change(dev, T, E, k, N, F, how, dtype):
    g = torch.Generator().manual_seed(T)
    x, weights, ids = torch.randn(T, N, generator=g).to(dtype), torch.randn(T, k, generator=g), _ids(g, T, E, k, how)
    stored, values = _weights(g, E, F, N, dtype, True, 0)
    out, off = oe.experts_ffn(x, ids, weights, *values, unit=UNIT[dtype], sums=sums)
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    got = blocks.ExpertsFfn().run(x.to(dev), ids.to(dev), weights.to(dev), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])
    assert_within(got, out, off * 1.01 + UNIT[dtype] * (out.abs() + off) + 2.0 ** -25, "experts")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M", [1, 3, 16, 30, 40, 100, 300])
@pytest.mark.parametrize("x4", [False, True])
def test_products_of_weights_that_the_type_holds_as_subnormals(dev, dtype, M, x4):
    """Every scale from that on whose values the type holds exactly (its least subnormal is half of 2^e): one value of K at a time, times
    a power of two that makes the product a normal number, exactly."""
    least, up = (-23, 10) if dtype == F16 else (-127, 20)
    scale = torch.arange(least, least + 16)
    N, K = 16, 512
    g = torch.Generator().manual_seed(M)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (scale + 127).to(torch.uint8).view(N, 1).repeat(1, K // 32)
    x = torch.zeros(M, K, dtype=dtype)
    at = torch.randint(0, K, (M,), generator=g)
    x[torch.arange(M), at] = 2.0 ** up
    values = oc.fp4_decode(codes, scales)
    assert torch.equal(values.to(dtype).double(), values) and bool((values.abs()[values != 0].min() < torch.finfo(dtype).smallest_normal))
    want = (values[:, at].t() * 2.0 ** up).to(dtype)
    assert torch.equal(want.double(), values[:, at].t() * 2.0 ** up)
    got = blocks.Fp4Matmul(quantize_x=x4).run(x.to(dev), codes.to(dev), scales.to(dev)).cpu()
    assert torch.equal(got, want)


@pytest.mark.parametrize("T", [1, 20, 300])
def test_experts_of_weights_that_the_type_holds_as_subnormals(dev, T):
    """Both products over 4-bit weights of every scale down to the last that fp16 holds: x and the hidden rows are large enough
    for results that count."""
    g = torch.Generator().manual_seed(T)
    E, k, N, F = 2, 1, 64, 96
    w = lambda *s: (torch.randint(0, 256, s[:-1] + (s[-1] // 2,), generator=g, dtype=torch.uint8),
                    (127 - 23 + torch.randint(0, 6, s[:-1] + (s[-1] // 32,), generator=g)).to(torch.uint8))
    stored = [w(E, F, N), w(E, F, N), w(E, N, F)]
    values = [oc.fp4_decode(*s) for s in stored]
    x = (4096 * torch.randn(T, N, generator=g)).half()
    ids, weights = _ids(g, T, E, k, "spread"), torch.full((T, k), 2.0 ** 14)
    out, off = oe.experts_ffn(x, ids, weights, *values, unit=UNIT[F16], sums=sums)
    assert float(out.abs().max()) > 100 * float(off.max())
    d = [t.to(dev) for s in stored for t in s]
    got = blocks.ExpertsFfn().run(x.to(dev), ids.to(dev), weights.to(dev), d[0], d[2], d[4], d[1], d[3], d[5])
    assert_within(got, out, off * 1.01 + UNIT[F16] * (out.abs() + off) + 2.0 ** -25, "experts")


@pytest.mark.parametrize("k", [65, 2 ** 31 - 1, 0, -1])
def test_choices_that_are_refused_take_no_memory(dev, k):
    z = torch.zeros(4096, 512, device=dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ext.TrinityError):
        blocks.Router(k).route(z)
    assert torch.cuda.max_memory_allocated() == before
    with pytest.raises(ext.TrinityError):
        blocks.Router(2).route(z.view(-1))
    assert torch.cuda.max_memory_allocated() == before


@pytest.mark.parametrize("w4", [False, True])
@pytest.mark.parametrize("prenorm", [False, True])
def test_routed_ffn_plan_is_its_parts(dev, w4, prenorm):
    """Logits in X's type, and an fp32 product in their place by the parts; no tokens; strided rows."""
    g = torch.Generator().manual_seed(12)
    T, E, k, N, F = 90, 16, 3, 256, 288
    stored, _ = _weights(g, E, F, N, BF16, w4, 0)
    d = [to_dev(t, dev) for s in stored for t in s]
    args = (d[0], d[2], d[4], d[1], d[3], d[5])
    x, wr = torch.randn(T, N, generator=g).bfloat16().to(dev), (0.1 * torch.randn(N, E, generator=g)).bfloat16().to(dev)
    plan = blocks.RoutedFfnPlan(k, prenorm=prenorm, eps=1e-5)
    got = plan.run(x, wr, *args)
    xn = x
    if prenorm:
        xn = torch.empty_like(x)
        ext.rmsnorm(x, None, xn, 1e-5)
    logits = torch.empty(T, E, dtype=BF16, device=dev)
    ext.matmul(xn, wr, None, logits)
    assert torch.equal(got, blocks.ExpertsFfn().run(xn, *blocks.Router(k).route(logits), *args))
    exact = xn.cpu().double() @ wr.cpu().double()
    ids, w = blocks.Router(k).route(exact.float().to(dev))  # (what a model with fp32 logits does)
    want, value = oe.route(exact.float(), top_k=k)
    assert torch.equal(ids.cpu().long(), want)
    assert_within(w, value, 2.0 ** -24 * value * 1.01, "weights")
    none = plan.run(x[:0], wr, *args)
    assert none.shape == (0, N) and none.dtype == BF16
    big = torch.full((T, N + 16), 3, dtype=BF16, device=dev)
    assert plan.run(x, wr, *args, out=big[:, 8:N + 8]).data_ptr() == big[:, 8:].data_ptr()
    assert torch.equal(big[:, 8:N + 8], got) and bool((big[:, :8] == 3).all()) and bool((big[:, N + 8:] == 3).all())


def _inside(t, left, right, fill):
    """The same values as columns of wider rows, between bytes that no call may read as its own."""
    rows = t.reshape(-1, t.shape[-1])
    wide = torch.full((rows.shape[0], left + t.shape[-1] + right), fill, dtype=t.dtype)
    wide[:, left:left + t.shape[-1]] = rows
    return wide.view(*t.shape[:-1], -1)[..., left:left + t.shape[-1]]


@pytest.mark.parametrize("M", [1, 4, 16, 30, 40, 100, 300])
@pytest.mark.parametrize("x4", [False, True])
def test_products_over_matrices_inside_larger_ones(dev, M, x4):
    """Weights, rows and scales whose rows are parts of wider ones, up to the last byte before what is not theirs (255: codes of -6, NaN)."""
    K, N = 1120, 72
    g = torch.Generator().manual_seed(M)
    w, ws = oc.fp4_encode(torch.randn(N, K, generator=g))
    x = torch.randn(M, K, generator=g).bfloat16()
    if x4:
        rows, xs = oc.fp4_encode(x)
        a = to_dev(_inside(rows, 16, 32, 255), dev), to_dev(_inside(xs, 3, 2, 255), dev)
        b = rows.to(dev), xs.to(dev)
    else:
        a, b = (to_dev(_inside(x, 8, 16, math.nan), dev), None), (x.to(dev), None)
    op = blocks.Fp4Matmul()
    want = op.run(b[0], w.to(dev), ws.to(dev), x_scales=b[1], dtype=BF16)
    got = op.run(a[0], to_dev(_inside(w, 32, 16, 255), dev), to_dev(_inside(ws, 5, 1, 255), dev), x_scales=a[1], dtype=BF16)
    assert bool(torch.isfinite(want).all()) and torch.equal(got, want)


@pytest.mark.parametrize("T", [1, 6, 90, 600])
@pytest.mark.parametrize("w4", [False, True])
def test_experts_over_matrices_inside_larger_ones(dev, T, w4):
    E, k, N, F = 5, 2, 544, 288
    g = torch.Generator().manual_seed(T)
    x, ids, weights = torch.randn(T, N, generator=g).bfloat16(), _ids(g, T, E, k, "few"), torch.rand(T, k, generator=g)
    stored, _ = _weights(g, E, F, N, BF16, w4, 0)
    plain = [(t.to(dev), None if s is None else s.to(dev)) for t, s in stored]
    inside = [(to_dev(_inside(t, 16, 32, 255 if w4 else math.nan), dev), to_dev(None if s is None else _inside(s, 3, 4, 255), dev)) for t, s in stored]
    op = blocks.ExpertsFfn()
    call = lambda x, d: op.run(x, ids.to(dev), weights.to(dev), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])
    want = call(x.to(dev), plain)
    assert bool(torch.isfinite(want).all())
    assert torch.equal(call(to_dev(_inside(x, 8, 24, math.nan), dev), inside), want)


@pytest.mark.parametrize("w4", [False, True])
def test_threads_share_objects_and_a_stream(dev, w4):
    E, k, N, F = 8, 2, 544, 1056
    g = torch.Generator().manual_seed(3)
    stored, _ = _weights(g, E, F, N, F16, w4, 0)
    d = [t.to(dev) if t is not None else None for s in stored for t in s]
    router, op = blocks.Router(k), blocks.ExpertsFfn()
    calls = [(torch.randn(T, N, generator=g).half().to(dev), torch.randn(T, E, generator=g).to(dev)) for T in (1, 20, 100, 700)]
    step = lambda x, z: op.run(x, *router.route(z), d[0], d[2], d[4], d[1], d[3], d[5])
    want = [step(*c) for c in calls]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(4) as threads:
        got = list(threads.map(lambda i: (i % 4, step(*calls[i % 4])), range(80)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
