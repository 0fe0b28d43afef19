"""Pins of oracle/experts.py, on the CPU: products entry by entry, routing by a search over all subsets, the experts' FFN against the
dense one."""
import itertools
import math

import pytest
import torch

from experts_util import sums
from oracle import cache as oc
from oracle import experts as oe


def test_products_entry_by_entry():
    g = torch.Generator().manual_seed(1)
    w, ws = oc.fp4_encode(torch.randn(8, 64, generator=g))
    x = torch.randn(3, 64, generator=g).half()
    xc, xs = oc.fp4_encode(x)
    for rows, scales in ((x, None), (xc, xs)):
        out, mag = oe.fp4_matmul(rows, w, ws, scales)
        for i in range(3):
            for j in range(8):
                terms = []
                for k in range(64):
                    code = lambda c, s, r: ((int(c[r, k // 2]) >> (4 * (k % 2))) & 15, math.ldexp(1.0, int(s[r, k // 32]) - 127))
                    value = lambda v: (-1 if v[0] >= 8 else 1) * oc.MAGNITUDES[v[0] % 8] * v[1]
                    terms.append(value(code(w, ws, j)) * (float(rows[i, k]) if scales is None else value(code(xc, xs, i))))
                assert abs(math.fsum(terms) - float(out[i, j])) <= 64 * 2.0 ** -53 * float(mag[i, j])
                assert abs(math.fsum(map(abs, terms)) - float(mag[i, j])) <= 64 * 2.0 ** -53 * float(mag[i, j])


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups,top_groups,group_top", [(1, 1, 1), (4, 2, 1), (4, 2, 2), (2, 1, 2)])
def test_routes_against_all_subsets(sigmoid, groups, top_groups, group_top):
    """The chosen experts have the largest sum of all allowed sets of that many, and groups likewise."""
    g = torch.Generator().manual_seed(groups + top_groups + group_top)
    T, E, k = 12, 8, 3
    z, bias = torch.randn(T, E, generator=g), 0.3 * torch.randn(E, generator=g)
    ids, weights = oe.route(z, bias, top_k=k, sigmoid=sigmoid, groups=groups, top_groups=top_groups, group_top=group_top,
                            renormalize=True, scale=2.0)
    s = torch.sigmoid(z.double()) if sigmoid else torch.softmax(z.double(), -1)
    c, size = s + bias.double(), E // groups
    for t in range(T):
        worth = lambda gs: sum(sum(sorted((float(c[t, e]) for e in range(gi * size, (gi + 1) * size)), reverse=True)[:group_top]) for gi in gs)
        stay = max(itertools.combinations(range(groups), top_groups), key=worth)
        allowed = [e for e in range(E) if e // size in stay]
        best = max(itertools.combinations(allowed, k), key=lambda es: sum(float(c[t, e]) for e in es))
        chosen = ids[t].tolist()
        assert set(chosen) == set(best) and all(c[t, a] >= c[t, b] for a, b in zip(chosen, chosen[1:]))
        assert torch.allclose(weights[t], 2.0 * s[t, ids[t]] / s[t, ids[t]].sum(), rtol=1e-14, atol=0)


def test_ties_go_to_the_lowest_index():
    ids, weights = oe.route(torch.tensor([[1.0, 2.0, 2.0, 1.0], [-math.inf] * 4]), top_k=3, renormalize=True)
    assert ids.tolist() == [[1, 2, 0], [0, 1, 2]] and weights[1].tolist() == [0, 0, 0]


def test_experts_against_the_dense_ffn():
    g = torch.Generator().manual_seed(2)
    T, E, N, F = 7, 3, 32, 64
    x = torch.randn(T, N, generator=g).half()
    gate, up = (torch.randn(E, F, N, generator=g).half() * 0.2 for _ in range(2))
    down = torch.randn(E, N, F, generator=g).half() * 0.2
    ids, weights = torch.tensor([[0, 2], [1, 1], [2, 0], [-1, 1], [3, 7], [1, 0], [2, -9]]), torch.randn(T, 2, generator=g)
    out, off = oe.experts_ffn(x, ids, weights, gate.double(), up.double(), down.double(), unit=2.0 ** -11, sums=sums)
    for t in range(T):
        want = torch.zeros(N, dtype=torch.float64)
        for i, e in enumerate(ids[t].tolist()):
            if 0 <= e < E:
                z = gate[e].double() @ x[t].double()
                want += float(weights[t, i]) * (down[e].double() @ (z / (1 + torch.exp(-z)) * (up[e].double() @ x[t].double())))
        assert torch.allclose(out[t], want, rtol=1e-12, atol=1e-12)
    assert bool((out[4] == 0).all()) and bool((off[4] == 0).all())
    # what fp32 and a 16-bit rounding of the hidden rows do stays within the bound
    for t in (0, 1, 2):
        got = torch.zeros(N)
        for i, e in enumerate(ids[t].tolist()):
            z = gate[e].float() @ x[t].float()
            h = (torch.nn.functional.silu(z) * (up[e].float() @ x[t].float())).half().float()
            got += weights[t, i] * (down[e].float() @ h)
        assert bool(((got.double() - out[t]).abs() <= off[t]).all())
