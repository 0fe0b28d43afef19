"""The plans of tri_fp4_matmul and tri_experts_ffn (csrc/group_tile.hip, group_stream.hip), on the CPU: the GPU tests meet every form
of their kernels, plans keep within their bounds, and the workspace that is asked for is what they use."""
import ctypes
import random

import pytest

import test_gpu_experts
import test_gpu_fp4
from trinity_amd import ext


class Plan(ctypes.Structure):
    _fields_ = [("bm", ctypes.c_int), ("parts", ctypes.c_int)]


def _fn(name, result):
    f = getattr(ext.lib(), name)
    f.restype = result
    return f


def rows_plan(M, K, N, x4):
    if not x4 and _fn("_ZN3tri18group_stream_takesEiib", ctypes.c_bool)(M, K, ctypes.c_bool(True)):
        return 16, _fn("_ZN3tri18group_stream_partsEiiii", ctypes.c_int)(M, K, N, 1)
    p = _fn("_ZN3tri15group_rows_planEiiib", Plan)(M, K, N, ctypes.c_bool(x4))
    return p.bm, p.parts


def experts_plan(T, k, E, N, F, w4):
    p = _fn("_ZN3tri12experts_planEiiiiib", Plan)(T * k, k, E, N, F, ctypes.c_bool(w4))
    return p.bm, p.parts


def test_products_meet_every_form():
    cases = list(test_gpu_fp4.FORMS) + [(M, K, N, x4) for M, K, N, *_ in test_gpu_fp4.PRODUCTS for x4 in (False, True)]
    seen, blocks = set(), set()
    for M, K, N, x4 in cases:
        bm, parts = rows_plan(M, K, N, x4)
        seen.add((x4, bm if bm > 16 else (1 if M <= 1 else (4 if M <= 4 else 16)), parts > 1))
        if bm == 256 and not x4:  # row blocks of 64 in a column's tiles
            blocks |= {4 if M >= 256 else 0, (M % 256 + 63) // 64}
    want = {(x4, bm, parts) for x4 in (False, True) for bm in (32, 64, 128, 256) for parts in (False, True)}
    want |= {(False, rows, parts) for rows in (1, 4, 16) for parts in (False, True)}
    assert not want - seen, sorted(want - seen)
    assert blocks >= {1, 2, 3, 4}


def test_experts_meet_every_form():
    seen = set()
    for T, E, k, N, F, how in test_gpu_experts.EXPERTS:
        for w4 in (False, True):
            bm, parts = experts_plan(T, k, E, N, F, w4)
            few = T * k <= 64
            if few and not w4 and min(N, F) >= 64:
                seen.add((w4, "strip", False))
            elif bm == 16:
                seen.add((w4, ("by choice", 1 if T == 1 else (4 if T <= 4 else 16)) if few else "in order", parts > 1))
            else:
                seen.add((w4, bm, parts > 1))
    want = {(False, "strip", False), (True, ("by choice", 1), False), (True, ("by choice", 4), False), (True, ("by choice", 16), False),
            (True, "in order", False)}
    want |= {(False, bm, parts) for bm in (64, 256) for parts in (False, True)}
    want |= {(True, bm, parts) for bm in (32, 128, 256) for parts in (False, True)}
    assert not want - seen, sorted(want - seen, key=str)


def test_plans_keep_their_bounds():
    rng = random.Random(3)
    for _ in range(3000):
        M, N, K = int(2 ** rng.uniform(0, 15)), 8 * int(2 ** rng.uniform(0, 12)), 32 * int(2 ** rng.uniform(0, 12))
        x4 = rng.random() < 0.5
        bm, parts = rows_plan(M, K, N, x4)
        assert bm in (16, 32, 64, 128, 256) and 1 <= parts
        if bm > 16:  # no part is empty, and parts of K are there to fill the GPU
            deep = -(-K // 256)
            per = -(-deep // parts)
            assert (parts - 1) * per < deep and (parts == 1 or per >= 2)
            cols = 256 if bm in (32, 256) else 128
            assert parts == 1 or -(-M // bm) * -(-N // cols) * parts <= 512
        need = ext.fp4_workspace_bytes(M, K, N, x4)
        assert need == (parts * M * N * 4 if parts > 1 else 0)


@pytest.mark.parametrize("seed", [1, 2])
def test_experts_plans_keep_their_bounds(seed):
    rng = random.Random(seed)
    for _ in range(2000):
        E = rng.choice((1, 2, 7, 8, 64, 512))
        k = rng.randint(1, min(E, 64))
        T = int(2 ** rng.uniform(0, 13))
        N, F = (32 * int(2 ** rng.uniform(0, 9)) for _ in range(2))
        n, most = T * k, 1
        for w4 in (False, True):
            bm, parts = experts_plan(T, k, E, N, F, w4)
            assert bm in ((16, 32, 128, 256) if w4 else (64, 256))
            deep = -(-F // (512 if bm == 16 else 256))
            assert (parts - 1) * -(-deep // parts) < deep
            assert bm == 16 or parts == 1 or -(-n // bm) * parts <= 1024
            most = max(most, parts)
        up = lambda b: -(-b // 256) * 256
        need = up(n * F * 2) + up(n * N * 4 * most) + up(n * 4) + up(16 * (1 + -(-n // 16) + min(E, n)))
        assert ext.experts_workspace_bytes(T, k, E, N, F) == need
