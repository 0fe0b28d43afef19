"""GPU parity of routing (tri_route) and of the experts' FFN (tri_experts_ffn) with oracle/experts.py, which computes in fp64.
Chosen experts are compared exactly, weights to an fp32 rounding, outputs within the bound of their roundings."""
import math

import pytest
import torch

import oracle
from cache_util import UNIT, assert_within
from experts_util import four_bit, sums, to_dev
from oracle import cache as oc
from oracle import experts as oe
from trinity_amd import blocks, ext

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# T, E, top_k, sigmoid, bias, groups, top_groups, group_top
ROUTES = [
    (1, 1, 1, False, False, 1, 1, 1), (1, 8, 2, False, False, 1, 1, 1), (33, 8, 8, True, False, 1, 1, 1), (5, 7, 3, False, True, 1, 1, 1),
    (70, 16, 4, True, True, 1, 1, 1), (9, 31, 31, False, False, 1, 1, 1), (300, 64, 6, False, False, 1, 1, 1),
    (17, 64, 64, True, False, 1, 1, 1), (40, 100, 10, True, True, 1, 1, 1), (200, 128, 8, False, True, 8, 3, 2),
    (200, 256, 8, True, True, 8, 4, 2), (64, 160, 6, False, False, 8, 3, 1), (50, 8, 2, True, True, 4, 2, 2),
    (50, 16, 3, False, False, 4, 2, 1), (20, 512, 16, True, False, 64, 5, 2), (30, 500, 5, False, True, 1, 1, 1),
]


@pytest.mark.parametrize("T,E,k,sigmoid,bias,groups,top_groups,group_top", ROUTES)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("renormalize,scale", [(True, 1.0), (False, 2.5), (True, -0.5)])
def test_route(dev, T, E, k, sigmoid, bias, groups, top_groups, group_top, dtype, renormalize, scale):
    g = torch.Generator().manual_seed(T * E + k)
    z = (1.5 * torch.randn(T, E + 3, generator=g)).to(dtype)
    if T > 4:
        z[1] = 0.25  # all the same: the lowest
        z[2, ::2] = -math.inf
        z[3] = torch.finfo(dtype).min
        z[4, : E // 2] = z[4, E - E // 2: E]
    b = 0.3 * torch.randn(E, generator=g) if bias else None
    kw = dict(sigmoid=sigmoid, groups=groups, top_groups=top_groups, group_top=group_top, renormalize=renormalize, scale=scale)
    want, w = oe.route(z[:, :E], b, top_k=k, **kw)
    kw["scores"] = "sigmoid" if kw.pop("sigmoid") else "softmax"
    op = blocks.Router(k, **kw)
    ids, weights = op.route(to_dev(z[:, :E], dev), None if b is None else b.to(dev))
    assert ids.dtype == torch.int32 and weights.dtype == F32
    assert torch.equal(ids.cpu().long(), want)
    assert_within(weights, w, 2.0 ** -24 * w.abs() * 1.01 + 2.0 ** -149, "weights")


@pytest.mark.parametrize("sigmoid", [False, True])
def test_route_without_a_choice(dev, sigmoid):
    """Rows of -inf only have weights of zero; a NaN or +inf leaves ids that are experts, each once."""
    z = torch.zeros(4, 12)
    z[0] = -math.inf
    z[1, 5], z[2, 3] = math.nan, math.inf
    for groups, top in ((1, 1), (3, 2)):
        ids, w = blocks.Router(6, scores="sigmoid" if sigmoid else "softmax", groups=groups, top_groups=top).route(z.to(dev))
        for row in ids.cpu().tolist():
            assert len(set(row)) == 6 and all(0 <= e < 12 for e in row)
        assert bool((w[0] == 0).all())
        assert bool(torch.isfinite(w[3]).all())


def test_route_many_tokens(dev):
    """More tokens than one launch has room for side by side, scores next to each other among them."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(20000, 64, generator=g).bfloat16()  # (many equal logits)
    ids, w = blocks.Router(4).route(z.to(dev))
    s = torch.softmax(z.double(), -1)
    order = s.sort(dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(ids.cpu().long(), order)
    want = s.gather(1, order)
    assert_within(w, want / want.sum(-1, keepdim=True), 2.0 ** -23, "weights")


def _ids(g, T, E, k, how):
    if how == "spread":
        return torch.rand(T, E, generator=g).argsort(-1)[:, :k].int()
    if how == "one":  # all tokens to the same experts
        return (torch.arange(k).int() + E - k).expand(T, k).contiguous()
    if how == "twice":  # an expert twice in a token
        return torch.randint(0, E, (T, 1), generator=g).int().expand(T, k).contiguous()
    ids = torch.rand(T, E, generator=g).argsort(-1)[:, :k].int()  # "few": some choices are none
    ids[torch.rand(T, k, generator=g) < 0.4] = -1
    ids[0] = torch.tensor([E, -5] + [2 ** 30] * k, dtype=torch.int32)[:k]
    return ids


# T, E, top_k, N, F, ids
EXPERTS = [
    (1, 8, 2, 256, 512, "spread"), (1, 4, 4, 288, 1120, "spread"), (1, 3, 2, 64, 96, "spread"), (1, 5, 3, 320, 256, "few"),
    (1, 5, 5, 256, 800, "twice"), (2, 8, 2, 544, 256, "spread"), (16, 8, 4, 256, 288, "spread"), (20, 6, 3, 256, 320, "one"),
    (21, 2, 3, 288, 256, "twice"), (9, 7, 6, 512, 256, "few"), (33, 8, 2, 96, 160, "spread"), (40, 6, 2, 256, 288, "few"),
    (13, 70, 6, 32, 64, "spread"), (50, 512, 2, 64, 32, "spread"), (100, 4, 2, 224, 416, "spread"), (130, 4, 2, 128, 96, "one"),
    (300, 5, 3, 160, 256, "spread"), (301, 9, 4, 96, 544, "few"), (520, 2, 2, 288, 160, "spread"), (600, 3, 2, 544, 352, "few"),
    (700, 2, 1, 96, 1056, "one"), (257, 1, 1, 64, 32, "spread"), (64, 3, 1, 64, 96, "twice"), (530, 2, 3, 32, 64, "twice"),
    # choices one by one, rows of one, four and sixteen; rows put in order (more than 64 choices)
    (1, 6, 2, 544, 1056, "spread"), (1, 9, 3, 1056, 512, "twice"), (4, 8, 3, 512, 544, "few"), (16, 8, 4, 1056, 512, "spread"),
    (13, 70, 6, 544, 512, "spread"), (5, 20, 16, 512, 544, "twice"), (40, 8, 2, 544, 800, "spread"), (15, 90, 40, 512, 576, "few"),
    # parts of K; two row blocks of four
    (50, 3, 2, 64, 1056, "spread"), (50, 2, 2, 96, 1088, "one"), (200, 2, 2, 64, 1056, "few"), (110, 2, 2, 96, 160, "one"),
]


def _weights(g, E, F, N, dtype, w4, layout):
    """gate, up, down and their scales on the CPU, and fp64 values."""
    res = []
    if w4:
        # experts' gate and up next to each other, as a checkpoint may have them; scales at odd addresses
        both, both_s = four_bit(g, E, 2 * F, N, std=N ** -0.5, shift=3 if layout else 0)
        down, down_s = four_bit(g, E, N, F, std=F ** -0.5, pad=1 if layout else 0)
        res = [(both[:, :F], both_s[:, :F]), (both[:, F:], both_s[:, F:]), (down, down_s)]
        if not layout:
            res = [(a.contiguous(), b.contiguous()) for a, b in res]
        return res, [oc.fp4_decode(a, b) for a, b in res]
    both = (torch.randn(E, 2 * F, N + 8 * layout, generator=g) * N ** -0.5).to(dtype)[:, :, :N]
    down = (torch.randn(E, N, F, generator=g) * F ** -0.5).to(dtype)
    if not layout:
        both = both.contiguous()
    ws = [both[:, :F], both[:, F:], down]
    return [(w, None) for w in ws], [w.double() for w in ws]


@pytest.mark.parametrize("T,E,k,N,F,how", EXPERTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("w4", [False, True])
def test_experts(dev, T, E, k, N, F, how, dtype, w4):
    g = torch.Generator().manual_seed(T + 31 * E + N + F)
    x = torch.randn(T, N + 8, generator=g).to(dtype)[:, :N]
    ids = _ids(g, T, E, k, how)
    weights = torch.randn(T, k, generator=g)
    stored, values = _weights(g, E, F, N, dtype, w4, T % 2)
    out, off = oe.experts_ffn(x, ids, weights, *values, unit=UNIT[dtype], sums=sums)
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    big = torch.full((T, N + 16), 3, dtype=dtype, device=dev)
    op = blocks.ExpertsFfn()
    args = (to_dev(x, dev), ids.to(dev), weights.to(dev), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])
    got = op.run(*args)
    tol = off * 1.01 + UNIT[dtype] * (out.abs() + off) + 2.0 ** -25
    assert_within(got, out, tol, "experts")
    op.run(*args, out=big[:, 8:N + 8])
    assert torch.equal(big[:, 8:N + 8], got)
    assert bool((big[:, :8] == 3).all()) and bool((big[:, N + 8:] == 3).all())


@pytest.mark.parametrize("T", [1, 5, 90, 600])
@pytest.mark.parametrize("w4", [False, True])
def test_rows_without_an_expert_are_zero_whatever_the_others_hold(dev, T, w4):
    """ids outside the experts count nothing: not their token's weights (NaN), nor what others make of NaN inputs."""
    g = torch.Generator().manual_seed(T)
    E, k, N, F = 4, 2, 288, 320
    stored, _ = _weights(g, E, F, N, BF16, w4, 0)
    x = torch.randn(T, N, generator=g).bfloat16()
    ids, weights = _ids(g, T, E, k, "spread"), torch.rand(T, k, generator=g)
    none = torch.arange(T) % 3 == 0
    ids[none] = -1
    weights[none] = math.nan
    x[none] = math.nan
    if T > 2:
        x[1] = math.inf
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    junk = torch.full((1 << 26,), 255, dtype=torch.uint8, device=dev)  # (the workspace is likely to be taken from here)
    del junk
    got = blocks.ExpertsFfn().run(x.to(dev), ids.to(dev), weights.to(dev), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1]).cpu()
    assert bool((got[none] == 0).all())
    other = ~none
    if T > 2:
        other[1] = False
        assert not bool(torch.isfinite(got[1]).any())
    assert bool(torch.isfinite(got[other]).all())


@pytest.mark.parametrize("T", [1, 7, 200])
@pytest.mark.parametrize("w4", [False, True])
def test_captured_and_replayed(dev, T, w4):
    """Routing and experts in one graph: which experts have rows changes between replays."""
    g = torch.Generator().manual_seed(T)
    E, k, N, F = 16, 3, 256, 320
    stored, _ = _weights(g, E, F, N, F16, w4, 0)
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    x, z = torch.zeros(T, N, dtype=F16, device=dev), torch.zeros(T, E, dtype=F16, device=dev)
    router, op = blocks.Router(k, scores="sigmoid"), blocks.ExpertsFfn()

    def step(x, z):
        ids, w = router.route(z)
        return ids, op.run(x, ids, w, d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])

    step(x, z)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # (two graphs that are alive at once share no workspace)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            res = step(x, z)
        graphs[-1].res = res
    for i in range(4):
        gi = torch.Generator().manual_seed(100 + i)
        nx, nz = torch.randn(T, N, generator=gi).half().to(dev), (2 * torch.randn(T, E, generator=gi)).half().to(dev)
        x.copy_(nx)
        z.copy_(nz)
        for graph in graphs:
            graph.replay()
        ids, out = step(nx, nz)
        torch.cuda.synchronize()
        for graph in graphs:
            assert torch.equal(graph.res[0], ids) and torch.equal(graph.res[1], out)


@pytest.mark.parametrize("w4", [False, True])
def test_two_streams_at_once(dev, w4):
    """Calls of one object on two streams, behind one another on the host and side by side on the GPU."""
    g = torch.Generator().manual_seed(8)
    E, k, N, F = 8, 2, 544, 1056
    stored, _ = _weights(g, E, F, N, BF16, w4, 0)
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    op, router, calls = blocks.ExpertsFfn(), blocks.Router(k), []
    for T in (1, 30, 200, 700):
        x, z = torch.randn(T, N, generator=g).bfloat16().to(dev), torch.randn(T, E, generator=g).to(dev)
        calls.append((x, z))

    def step(x, z):
        return op.run(x, *router.route(z), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])

    want = [step(*c) for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, c in enumerate(calls):
            for s in (streams[i % 2], streams[1 - i % 2]):
                with torch.cuda.stream(s):
                    got.append((i, step(*c)))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])


def test_results_do_not_depend_on_timing(dev):
    """Rows of an expert are taken in the order of the tokens: the same call has the same bits."""
    g = torch.Generator().manual_seed(2)
    T, E, k, N, F = 500, 8, 2, 256, 512
    stored, _ = _weights(g, E, F, N, BF16, False, 0)
    a = (torch.randn(T, N, generator=g).bfloat16().to(dev), _ids(g, T, E, k, "spread").to(dev), torch.rand(T, k, generator=g).to(dev))
    w = [s[0].to(dev) for s in stored]
    op = blocks.ExpertsFfn()
    first = op.run(*a, *w)
    for _ in range(5):
        assert torch.equal(op.run(*a, *w), first)


@pytest.mark.parametrize("T", [1, 6, 150])
@pytest.mark.parametrize("w4", [False, True])
def test_routed_ffn_plan(dev, T, w4):
    """The FFN half of a layer: norm, router, routing and experts, as they are used together."""
    g = torch.Generator().manual_seed(T)
    E, k, N, F = 8, 2, 256, 288
    stored, values = _weights(g, E, F, N, F16, w4, 0)
    x, wr = torch.randn(T, N, generator=g).half(), (0.1 * torch.randn(N, E, generator=g)).half()
    nw, bias = (1 + 0.1 * torch.randn(N, generator=g)).half(), 0.1 * torch.randn(E, generator=g)
    plan = blocks.RoutedFfnPlan(k, scores="sigmoid", prenorm=True, eps=1e-5, scale=2.0)
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    got = plan.run(x.to(dev), wr.to(dev), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1], bias=bias.to(dev), norm_w=nw.to(dev))
    # the parts one by one, on what the part before left
    xn = torch.empty(T, N, dtype=F16, device=dev)
    ext.rmsnorm(x.to(dev), nw.to(dev), xn, 1e-5)
    logits = torch.empty(T, E, dtype=F16, device=dev)
    ext.matmul(xn, wr.to(dev), None, logits)
    assert_within(xn, oracle.rmsnorm(x, nw, 1e-5), 4e-3, "norm")
    ids, w = oe.route(logits, bias, top_k=k, sigmoid=True, scale=2.0)
    out, off = oe.experts_ffn(xn, ids, w, *values, unit=UNIT[F16], sums=sums)
    # (the weights' own fp32 rounding: 2^-24 of the output's magnitude, far below `off`)
    assert_within(got, out, off * 1.05 + UNIT[F16] * (out.abs() + off) + 2.0 ** -25, "routed FFN")


@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("w4", [False, True])
def test_routed_ffn_plan_captured(dev, T, w4):
    g = torch.Generator().manual_seed(T)
    E, k, N, F = 16, 4, 544, 576
    stored, _ = _weights(g, E, F, N, BF16, w4, 0)
    d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
    wr = (0.1 * torch.randn(N, E, generator=g)).bfloat16().to(dev)
    plan = blocks.RoutedFfnPlan(k, groups=4, top_groups=2, prenorm=True, eps=1e-5)
    x = torch.zeros(T, N, dtype=BF16, device=dev)
    step = lambda x: plan.run(x, wr, d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])
    step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for i in range(4):
        new = torch.randn(T, N, generator=g).bfloat16().to(dev)
        x.copy_(new)
        graph.replay()
        eager = step(new)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_a_few_choices_of_one_expert_more_often_than_tokens(dev):
    """More rows of an expert than tokens, more than a launch for few rows holds at a time."""
    g = torch.Generator().manual_seed(6)
    for T, E, k, N, F in ((1, 2, 40, 512, 544), (3, 3, 64, 544, 512), (2, 100, 64, 512, 544)):
        ids = torch.randint(0, 2, (T, k), generator=g).int()
        for w4 in (False, True):
            stored, values = _weights(g, E, F, N, F16, w4, 0)
            x, weights = torch.randn(T, N, generator=g).half(), torch.randn(T, k, generator=g)
            out, off = oe.experts_ffn(x, ids, weights, *values, unit=UNIT[F16], sums=sums)
            d = [(to_dev(a, dev), to_dev(b, dev)) for a, b in stored]
            got = blocks.ExpertsFfn().run(x.to(dev), ids.to(dev), weights.to(dev), d[0][0], d[1][0], d[2][0], d[0][1], d[1][1], d[2][1])
            assert_within(got, out, off * 1.01 + UNIT[F16] * (out.abs() + off) + 2.0 ** -25, "experts")


def test_empty(dev):
    g = torch.Generator().manual_seed(1)
    w = [s[0].to(dev) for s in _weights(g, 4, 64, 96, F16, False, 0)[0]]
    x, ids, p = torch.empty(0, 96, dtype=F16, device=dev), torch.empty(0, 2, dtype=torch.int32, device=dev), torch.empty(0, 2, device=dev)
    assert blocks.ExpertsFfn().run(x, ids, p, *w).shape == (0, 96)
    ids, p = blocks.Router(2).route(torch.empty(0, 4, device=dev))
    assert ids.shape == p.shape == (0, 2)
