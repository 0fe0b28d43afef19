"""Inputs and error bounds of the cache tests."""
import math

import torch

from oracle import cache as oc

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def make_caches(seed, B, Hkv, rows, D, dtype, four_bit, layout="bhld"):
    """Two caches of normal values (k with channels of different size) and, for 4 bits, their scales; fp64 values."""
    g = torch.Generator().manual_seed(seed)
    res = []
    for which in range(2):
        x = torch.randn(B, Hkv, rows, D, generator=g)
        if which == 0:
            x = x * torch.exp(0.5 * torch.randn(Hkv, 1, D, generator=g))
        x = x.to(dtype)
        if four_bit:
            codes, scales = oc.fp4_encode(x)
            res.append((_lay(codes, layout), _lay(scales, layout)))
        else:
            res.append((_lay(x, layout), None))
    return res[0][0], res[1][0], res[0][1], res[1][1]


def _lay(t, layout):
    """The same values, rows of one position next to one another ("blhd") or heads apart ("bhld")."""
    return t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "blhd" else t


def values(cache, scales):
    return cache.double() if scales is None else oc.fp4_decode(cache, scales)


def attention_tolerance(q, k, v, lens, mag, out, dtype, *, n_q_heads, scale):
    """Elementwise bound of |kernel - exact|: probabilities and the result rounded to `dtype` (half a step each, the former
    weighted with |v|), fp32 scores (D products, of a row's largest sum of magnitudes), fp32 sums over the keys (sixteen a
    matrix instruction), and probabilities under fp16's normal range (half its least step each, the largest being at
    least one)."""
    B, Hkv, _, D = k.shape
    n = max(max(lens), 1)
    u = UNIT[dtype]
    qa = q.double().abs().amax().item()
    ka = max([k[b, :, :m].nan_to_num(0, 0, 0).abs().sum(-1).amax().item() for b, m in enumerate(lens) if m > 0] + [0.0])
    va = max([v[b, :, :m].nan_to_num(0, 0, 0).abs().amax().item() for b, m in enumerate(lens) if m > 0] + [0.0])
    e_s = (D + 16) * 2.0 ** -24 * scale * qa * ka
    e_l = (n / 16 + 64) * 2.0 ** -24
    tiny = n * 2.0 ** -25 * va if dtype == torch.float16 else 0.0
    return (u * (mag + out.abs()) + (2 * e_s + 2 * e_l) * mag + tiny) * 1.01 + 2.0 ** -24, e_s + e_l


def assert_within(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), what + ": values that are no numbers"
    off = (got - want).abs()
    bad = off > tol
    if bool(bad.any()):
        at = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError("%s: %d of %d out of tolerance, the first at %s: got %g, want %g, tolerance %g"
                             % (what, int(bad.sum()), got.numel(), at, got[at], want[at], (tol[at] if torch.is_tensor(tol) else tol)))
