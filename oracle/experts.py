"""Products over 4-bit weights, routing to experts and the experts' FFN, in fp64 (the reference has no counterpart: these
functions are the definition).  tests/test_experts_oracle.py pins them: products against decoded matrices entry by entry,
routing against a search over all subsets of experts, the FFN against a dense one per token.  4-bit matrices are
those of oracle/cache.py."""
import math

import torch

from .cache import fp4_decode


def fp4_matmul(x, w, w_scales, x_scales=None):
    """fp64 x . w^T and the sums of |x| . |w|^T; x values, or codes with x_scales."""
    x = x.detach().cpu().double() if x_scales is None else fp4_decode(x, x_scales)
    w = fp4_decode(w, w_scales)
    return x @ w.t(), x.abs() @ w.abs().t()


def route(logits, bias=None, *, top_k, sigmoid=False, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    """ids int64 and weights fp64 [T, top_k]."""
    z = logits.detach().cpu().double()
    T, E = z.shape
    ids, weights = torch.empty(T, top_k, dtype=torch.int64), torch.empty(T, top_k, dtype=torch.float64)
    for t in range(T):
        row = z[t].tolist()
        if sigmoid:
            s = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in row]
        elif max(row) == -math.inf:
            s = [0.0] * E
        else:
            p = [math.exp(v - max(row)) for v in row]
            s = [v / math.fsum(p) for v in p]
        c = [v + (float(bias[e]) if bias is not None else 0.0) for e, v in enumerate(s)]
        size = E // groups
        score = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_top]) for g in range(groups)]
        best = sorted(range(groups), key=lambda g: (-score[g], g))[:top_groups]
        order = sorted((e for e in range(E) if e // size in best), key=lambda e: (-c[e], e))[:top_k]
        total = math.fsum(s[e] for e in order)
        ids[t] = torch.tensor(order)
        for i, e in enumerate(order):
            weights[t, i] = (s[e] / total if total else 0.0) * scale if renormalize else s[e] * scale
    return ids, weights


def experts_ffn(x, ids, weights, gate, up, down, *, unit, sums):
    """fp64 out [T, N], and a bound of a kernel's error: hidden rows rounded with `unit` relative, a product over K values off
    by at most sums(K) of its sum of magnitudes.  gate, up [E, F, N] and down [E, N, F]: fp64 values."""
    x, weights = x.detach().cpu().double(), weights.detach().cpu().double()
    T, N = x.shape
    E, F = gate.shape[0], gate.shape[1]
    out, off = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    total = torch.zeros(T, N, dtype=torch.float64)
    for t in range(T):
        for i, e in enumerate(ids[t].tolist()):
            if not 0 <= e < E:
                continue
            g, u = gate[e] @ x[t], up[e] @ x[t]
            dg, du = sums(N) * (gate[e].abs() @ x[t].abs()), sums(N) * (up[e].abs() @ x[t].abs())
            s = g * torch.sigmoid(g)
            h = s * u
            # silu has a slope of at most 1.1, and is computed to 2^-20
            dh = 1.1 * dg * (u.abs() + du) + s.abs() * du + h.abs() * (unit * 1.01 + 2.0 ** -20) + 2.0 ** -25
            y = down[e] @ h
            mag = down[e].abs() @ (h.abs() + dh)
            w = abs(weights[t, i])
            out[t] += weights[t, i] * y
            off[t] += w * (down[e].abs() @ dh + sums(F) * mag)
            total[t] += w * mag
    return out, off + (ids.shape[1] + 1) * 2.0 ** -24 * total
