"""What the GPU tests of attention over caches of several sequences meet, on the CPU: every form of the plans with every kind of mask,
and that their bounds see a single key."""

import pytest
import torch

import test_gpu_cache
from cache_cases import MASKED, PLANTED, masks, planted, planted_tolerance
from cache_util import assert_within
from oracle import cache as oc
from test_cache_plans import plan


def test_every_form_meets_every_mask():
    seen = set()
    for case in test_gpu_cache.ATTN + MASKED:
        B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks = case
        for four_bit in (False, True):
            p = plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit)
            seen |= {(D, four_bit, p.nt, p.ways, min(p.runs, 2), m) for m in masks(*case)}
    want = {(D, f, nt, ways, runs, m) for D in (64, 128) for f in (False, True) for runs in (1, 2)
            for nt, ways in ((1, 1), (2, 1), (0, 1), (0, 2)) if f or nt < 2
            for m in ("window", "sinks", "padding", "window+padding", "all keys", "all keys+padding")}
    assert not want - seen, sorted(want - seen)


def test_long_lists_meet_every_form_in_runs():
    seen = set()
    for B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks in PLANTED:
        for four_bit in (False, True):
            p = plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit)
            seen.add((D, four_bit, p.nt, min(p.runs, 2), window > 0))
    want = {(D, f, nt, 2, w) for D in (64, 128) for f in (False, True) for nt in ((0, 1, 2) if f else (0, 1)) for w in (False, True)}
    assert not want - seen, sorted(want - seen)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("case", [PLANTED[1], PLANTED[2], PLANTED[8]], ids=str)
def test_one_missing_or_doubled_key_is_seen(case, dtype, four_bit):
    """The mistake is planted in the oracle: its output without a planted key, and with one twice, is out of the bound."""
    B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks = case
    p = plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit)
    q, c, k, v, n, at = planted(case, dtype, four_bit, 32 if p.nt else 64, p.runs)
    kw = dict(n_q_heads=Hq, causal=causal, window=window, sinks=sinks)
    want, lse, mag = oc.cache_attention(q, k, v, n, **kw)
    tol, tol_lse = planted_tolerance(D, n, dtype, mag, want)
    last = oc.visible(n[0], S, causal, window, sinks)[-1]
    keys = [x for x in at[0] if last[x]]
    assert len(keys) > 20
    for key in keys[:: len(keys) // 4] + [keys[-1]]:
        off = v.clone()
        off[0, 0, key] = 0  # (its weight in the sum is one of many: the value alone)
        with pytest.raises(AssertionError):
            assert_within(oc.cache_attention(q, k, off, n, **kw)[0], want, tol, "missing")
        off[0, 0, key] = 2 * v[0, 0, key]
        with pytest.raises(AssertionError):
            assert_within(oc.cache_attention(q, k, off, n, **kw)[0], want, tol, "twice")
