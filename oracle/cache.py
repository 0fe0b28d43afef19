"""Caches of several sequences and attention over them, in fp64 (the reference has no counterpart: these functions are
the definition).  tests/test_cache_oracle.py pins them: every 16-bit value's code against a search over the sixteen, the
block exponent against its defining inequality, attention against loops over single scores and against
F.scaled_dot_product_attention."""
import math

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK, MIN_EXP, NAN_BYTE = 32, -110, 255


def fp4_encode(x):
    """Codes [..., D / 2] and scale bytes [..., D / 32] (uint8) of rows x [..., D]."""
    blk = x.detach().cpu().double().reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    amax = blk.abs().amax(-1)
    bad = ~torch.isfinite(blk).all(-1)
    amax = torch.where(bad, 0.0, amax)
    mant, e = torch.frexp(amax)  # amax = mant 2^e, mant in [0.5, 1): 7 * 2^(e - 3) is 0.875 * 2^e
    e = torch.where(mant >= 0.875, e - 2, e - 3)
    e = torch.where(amax == 0, torch.full_like(e, MIN_EXP), e).clamp(min=MIN_EXP)
    y = blk / torch.ldexp(torch.ones_like(amax), e)[..., None]
    a = y.abs()
    # steps of a half below 2, of one below 4, of two above; torch.round takes ties to even, which are the even codes
    index = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2).clamp(max=3) + 4))
    code = index.long() + 8 * torch.signbit(y).long()
    code = torch.where(bad[..., None], 0, code).reshape(x.shape)
    scales = torch.where(bad, NAN_BYTE, e.long() + 127)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scales.to(torch.uint8)


def fp4_decode(codes, scales):
    """fp64 rows [..., D]."""
    codes, scales = codes.detach().cpu().long(), scales.detach().cpu().long()
    code = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    mag = torch.tensor(MAGNITUDES, dtype=torch.float64)[code % 8]
    val = torch.where(code >= 8, -mag, mag).reshape(*code.shape[:-1], code.shape[-1] // BLOCK, BLOCK)
    unit = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales - 127)
    unit = torch.where(scales == NAN_BYTE, math.nan, unit)
    return (val * unit[..., None]).flatten(-2)


def visible(n, seq, causal, window, sinks):
    """[seq, n] truth values: whether token i of a sequence of n keys sees key j (padding sees nothing)."""
    pos = torch.arange(n - seq, n)[:, None]
    key = torch.arange(n)[None]
    seen = (pos >= 0) & (key >= 0)
    if causal:
        seen = seen & (key <= pos)
    if window > 0:
        seen = seen & ((key > pos - window) | (key < sinks))
    return seen


def cache_attention(q, k, v, lens, *, n_q_heads, scale=None, causal=True, window=0, sinks=0):
    """fp64: out [B * S, Hq * D], lse [B, Hq, S] and the sums of p * |v| like out (what bounds rounding errors of p).
    q [B * S, Hq * D]; k, v [B, Hkv, rows, D]; lens: a list."""
    B, Hkv, _, D = k.shape
    S, g = q.shape[0] // B, n_q_heads // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q = q.detach().cpu().double().view(B, S, n_q_heads, D)
    out = torch.zeros(B, S, n_q_heads, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((B, n_q_heads, S), -math.inf, dtype=torch.float64)
    for b, n in enumerate(lens):
        seen = visible(n, S, causal, window, sinks)
        some = seen.any(1)
        if not some.any():
            continue
        used = seen.any(0)  # (what no token sees is not looked at: it may be anything)
        for hk in range(Hkv):
            kk, vv = k[b, hk, :n].double()[used], v[b, hk, :n].double()[used]
            s = torch.matmul(q[b, some, hk * g:(hk + 1) * g].transpose(0, 1), kk.t()) * scale
            s = torch.where(seen[some][:, used], s, -math.inf)
            p = torch.softmax(s, -1)
            lse[b, hk * g:(hk + 1) * g, some] = torch.logsumexp(s, -1)
            out[b, some, hk * g:(hk + 1) * g] = torch.matmul(p, vv).transpose(0, 1)
            mag[b, some, hk * g:(hk + 1) * g] = torch.matmul(p, vv.abs()).transpose(0, 1)
    return out.view(B * S, -1), lse, mag.view(B * S, -1)
