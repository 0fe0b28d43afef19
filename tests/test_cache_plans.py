"""The plans of tri_cache_attention (csrc/cache_attn.hip: cache_plan), on the CPU: the GPU tests meet every form of its kernels,
plans keep within their bounds, and the scratch that is asked for is what the plan uses."""
import ctypes
import random

import pytest

import test_gpu_cache
from trinity_amd import ext


class Plan(ctypes.Structure):
    _fields_ = [("nt", ctypes.c_int), ("ways", ctypes.c_int), ("runs", ctypes.c_int), ("nwg", ctypes.c_int64)]


def plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit):
    f = ext.lib()._ZN3tri10cache_planEiiiiiiiib
    f.restype = Plan
    return f(B, S, Hq, Hkv, D, kv_len, window, sinks, ctypes.c_bool(four_bit))


def test_gpu_cases_meet_every_form():
    seen = set()
    for B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks in test_gpu_cache.ATTN:
        for four_bit in (False, True):
            p = plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit)
            seen.add((D, four_bit, p.nt, p.ways, min(p.runs, 2)))
    want = {(D, f, nt, ways, runs) for D in (64, 128) for f in (False, True) for runs in (1, 2)
            for nt, ways in ((1, 1), (2, 1), (0, 1), (0, 2)) if f or nt < 2}
    assert not want - seen, sorted(want - seen)


@pytest.mark.parametrize("four_bit", [False, True])
def test_plans_keep_their_bounds(four_bit):
    rng = random.Random(7)
    for _ in range(3000):
        D, Hkv = rng.choice((64, 128)), rng.choice((1, 2, 4, 8, 32))
        Hq, B = Hkv * rng.choice((1, 2, 4, 7, 71)), rng.choice((1, 1, 2, 3, 8, 33))
        S, kv_len = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 20))
        window = rng.choice((0, 0, int(2 ** rng.uniform(0, 14)), 1 << 30))
        sinks = rng.choice((0, 4, 100, 1 << 30))
        p = plan(B, S, Hq, Hkv, D, kv_len, window, sinks, four_bit)
        rows = S * (Hq // Hkv)
        keys = min(kv_len, S + window + sinks) if window else kv_len
        most = 32 if four_bit and B * Hkv * keys >= 1 << 17 else 16
        assert p.nt == ((rows + 15) // 16 if rows <= most else 0) and p.ways in (1, 2) and 1 <= p.runs <= 64
        assert p.nwg == (B * Hkv if p.nt else -(-rows // 128) * B * Hkv)
        assert p.runs == 1 or p.nwg * p.runs <= 2048
        assert p.ways == 1 or (p.nt == 0 and p.nwg * p.runs <= 256)
        if B * S * Hq * (D // 8) >= (1 << 31) - 4096:  # refused
            continue
        params = ext.cache_params(B, Hkv, D, S, kv_len, n_q_heads=Hq, window=window, sinks=sinks)
        need = ext.cache_scratch_bytes(params, four_bit)
        assert need == (p.runs * B * S * Hq * (D + 2) * 4 if p.runs > 1 else 0)
