"""Pins of oracle/cache.py, on the CPU: 4-bit blocks by their definition, attention by loops and by torch's own."""
import math

import pytest
import torch

from oracle import cache as oc


def _nearest(y):
    """Index of the magnitude nearest to |y|, ties to the even index."""
    d = (torch.tensor(oc.MAGNITUDES, dtype=torch.float64) - y.abs()[..., None]).abs()
    best = d.amin(-1, keepdim=True)
    index = torch.arange(8).expand_as(d)
    among = torch.where(d == best, index, 99)
    even = torch.where((d == best) & (index % 2 == 0), index, 99).amin(-1)
    return torch.where(even < 99, even, among.amin(-1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_value_gets_the_nearest_code(dtype):
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype)
    x = x[torch.isfinite(x)]
    x = torch.cat((x, x[: -len(x) % 32]))
    for rows in (x.view(-1, 32), x.view(32, -1).t().contiguous()):
        codes, scales = oc.fp4_encode(rows)
        e = scales.long()[:, 0] - 127
        amax = rows.double().abs().amax(1)
        unit = torch.ldexp(torch.ones(len(e), dtype=torch.float64), e)
        assert bool((amax < 7 * unit).all()) and bool(((e == oc.MIN_EXP) | (amax >= 3.5 * unit)).all())
        code = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
        assert torch.equal(code % 8, _nearest(rows.double() / unit[:, None]))
        assert torch.equal(code >= 8, torch.signbit(rows))
        back = oc.fp4_decode(codes, scales)
        assert bool(((back - rows.double()).abs() <= unit[:, None]).all())  # half the widest step of two


def test_blocks_that_are_not_numbers():
    x = torch.ones(4, 64)
    x[0, 3], x[1, 40], x[2, 63] = math.inf, math.nan, -math.inf
    codes, scales = oc.fp4_encode(x.half())
    assert scales.tolist() == [[255, 125], [125, 255], [125, 255], [125, 125]]
    back = oc.fp4_decode(codes, scales)
    assert torch.isnan(back[0, :32]).all() and torch.equal(back[0, 32:], torch.ones(32, dtype=torch.float64))


@pytest.mark.parametrize("causal,window,sinks", [(False, 0, 0), (True, 0, 0), (True, 3, 0), (True, 3, 2), (True, 1, 1)])
def test_attention_by_loops(causal, window, sinks):
    g = torch.Generator().manual_seed(3)
    B, S, Hq, Hkv, D, lens = 4, 4, 4, 2, 64, [9, 4, 2, 0]
    q = torch.randn(B * S, Hq * D, generator=g)
    k, v = (torch.randn(B, Hkv, 10, D, generator=g) for _ in range(2))
    k[3], v[0, :, 9:] = math.nan, math.nan
    out, lse, mag = oc.cache_attention(q, k, v, lens, n_q_heads=Hq, causal=causal, window=window, sinks=sinks)
    for b, n in enumerate(lens):
        for i in range(S):
            for h in range(Hq):
                pos = n - S + i
                keys = [] if pos < 0 else [j for j in range(n) if not causal or (j <= pos and (window == 0 or j > pos - window or j < sinks))]
                got = out[b * S + i, h * D:(h + 1) * D]
                if not keys:
                    assert not got.any() and lse[b, h, i] == -math.inf
                    continue
                s = [float(q[b * S + i, h * D:(h + 1) * D].double() @ k[b, h // 2, j].double()) / 8 for j in keys]
                e = [math.exp(x) for x in s]
                want = sum(w * v[b, h // 2, j].double() for w, j in zip(e, keys)) / sum(e)
                assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
                assert abs(float(lse[b, h, i]) - math.log(sum(e))) < 1e-12
                assert bool((mag[b * S + i, h * D:(h + 1) * D] >= got.abs() - 1e-12).all())


def test_attention_against_torch():
    g = torch.Generator().manual_seed(4)
    S, H, D = 37, 3, 64
    q = torch.randn(S, H * D, generator=g).double()
    k, v = (torch.randn(1, H, S, D, generator=g).double() for _ in range(2))
    out = oc.cache_attention(q, k, v, [S], n_q_heads=H)[0]
    want = torch.nn.functional.scaled_dot_product_attention(q.view(1, S, H, D).transpose(1, 2), k, v, is_causal=True)
    assert torch.allclose(out, want[0].transpose(0, 1).reshape(S, -1), rtol=1e-12, atol=1e-12)
