"""GPU parity of attention over caches of several sequences: every form of its kernels with every kind of mask, and lists in which
each key at a border of tiles, waves and runs is seen by itself."""
import math

import pytest
import torch

import test_cache_plans
from cache_cases import MASKED, PLANTED, planted, planted_tolerance
from oracle import cache as oc
from test_gpu_cache import _case, _check, _lens
from trinity_amd import blocks

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("case", MASKED, ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("four_bit", [False, True])
def test_masks(dev, case, dtype, four_bit):
    B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks = case
    q, c, ln, *ref = _case(dev, *case, dtype, four_bit)
    op = blocks.CachedAttention(Hq, Hkv, D, causal=causal, window=window, sinks=sinks)
    out = torch.full((B * S, Hq * D), math.nan, dtype=dtype, device=dev)
    got, lse = op.attend(q, c[0], c[1], c[2], c[3], lens=ln, kv_len=kv_len, out=out, want_lse=True)
    _check(got, lse, *ref)


@pytest.mark.parametrize("case", PLANTED, ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("four_bit", [False, True])
def test_every_key_counts_once(dev, case, dtype, four_bit):
    B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks = case
    p = test_cache_plans.plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit)
    q, c, k, v, n, at = planted(case, dtype, four_bit, 32 if p.nt else 64, p.runs)
    want, lse, mag = oc.cache_attention(q, k, v, n, n_q_heads=Hq, causal=causal, window=window, sinks=sinks)
    tol, tol_lse = planted_tolerance(D, n, dtype, mag, want)
    op = blocks.CachedAttention(Hq, Hkv, D, causal=causal, window=window, sinks=sinks)
    got = op.attend(q.to(dev), *[None if x is None else x.to(dev) for x in c], lens=_lens(lens, dev), kv_len=kv_len, want_lse=True)
    _check(*got, want, lse, tol, tol_lse)


@pytest.mark.parametrize("prenorm,qknorm", [(False, False), (True, True)])
def test_block_of_no_tokens(dev, prenorm, qknorm):
    plan = blocks.CachedAttentionPlan(4, 2, 64, prenorm=prenorm, qknorm=qknorm)
    x, w = torch.zeros(0, 128, dtype=F16, device=dev), [torch.ones(128, 64 * h, dtype=F16, device=dev) for h in (4, 2, 2)]
    c = [torch.ones(3, 2, 8, 64, dtype=F16, device=dev) for _ in range(2)]
    out = plan.run(x, *w, None, *c, norm_w=torch.ones(128, dtype=F16, device=dev) if prenorm else None)
    assert out.shape == (0, 256) and bool((c[0] == 1).all())
