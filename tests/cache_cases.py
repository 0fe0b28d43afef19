"""Cases of attention over caches of several sequences: each of the plans' forms (csrc/cache_attn.hip: cache_plan) with each kind
of mask, found by a search over small sizes, and long lists whose keys are seen one by one.

A case: B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks."""
import math

import torch

from cache_util import UNIT
from oracle import cache as oc

MASKED = [
    (2, 3, 2, 1, 64, 13, 4, [4, 1], False, 0, 0),
    (2, 2, 10, 2, 128, 6, 2, [2, 1], False, 0, 0),
    (2, 5, 4, 1, 64, 6, 6, [6, 3], False, 0, 0),
    (3, 4, 7, 1, 128, 14, 5, [5, 4, 2], False, 0, 0),
    (2, 19, 1, 1, 64, 288, 282, [282, 18], True, 110, 70),
    (2, 2, 1, 1, 64, 662, 662, [662, 1], False, 0, 0),
    (2, 6, 3, 1, 128, 207, 202, [202, 5], False, 0, 0),
    (2, 2, 2, 1, 128, 648, 644, [644, 1], False, 0, 0),
    (4, 82, 5, 1, 64, 336, 330, [330, 39, 297, 6], False, 0, 0),
    (3, 9, 120, 24, 64, 964, 964, [964, 601, 2], False, 0, 0),
    (5, 153, 3, 3, 128, 362, 360, [360, 103, 345, 213, 123], True, 170, 37),
    (2, 6, 192, 64, 128, 1055, 1052, [1052, 3], False, 0, 0),
    (2, 6, 192, 64, 64, 1031, 1029, [1029, 1], False, 0, 0),
    (5, 12, 128, 64, 64, 423, 418, [418, 38, 373, 321, 1], True, 399, 0),
    (2, 3, 10, 2, 64, 54, 54, [54, 1], True, 42, 0),
    (2, 7, 2, 1, 128, 93, 92, [92, 3], True, 48, 3),
    (2, 7, 3, 1, 128, 94, 92, [92, 6], True, 76, 0),
    (2, 2, 1, 1, 64, 880, 874, [874, 1], True, 793, 3),
    (2, 2, 1, 1, 128, 955, 951, [951, 1], True, 719, 3),
    (4, 19, 24, 3, 64, 382, 375, [375, 213, 158, 6], True, 302, 5),
    (3, 6, 144, 48, 128, 1061, 1054, [1054, 268, 1], True, 996, 3),
    (5, 8, 80, 16, 64, 1086, 1083, [1083, 720, 417, 388, 7], True, 1007, 5),
    (5, 5, 224, 32, 128, 841, 836, [836, 155, 375, 91, 3], False, 0, 0),
    (3, 3, 8, 1, 64, 144, 143, [143, 142, 1], True, 108, 5),
    (2, 3, 448, 64, 128, 1086, 1082, [1082, 2], True, 987, 37),
    (5, 9, 64, 32, 64, 1065, 1064, [1064, 869, 749, 362, 2], True, 1018, 0),
    (2, 3, 1, 1, 64, 220, 219, [219, 2], True, 10, 5),
    (3, 6, 2, 1, 128, 91, 84, [84, 3, 1], True, 39, 0),
    (3, 12, 2, 1, 128, 77, 77, [77, 26, 1], True, 50, 3),
    (2, 10, 2, 1, 64, 295, 287, [287, 3], False, 0, 0),
    (2, 5, 1, 1, 64, 863, 856, [856, 1], True, 836, 0),
    (2, 9, 2, 1, 128, 290, 282, [282, 7], True, 153, 0),
    (2, 8, 1, 1, 128, 831, 831, [831, 4], True, 720, 0),
    (3, 25, 16, 16, 64, 387, 379, [379, 63, 20], True, 325, 0),
    (3, 12, 192, 48, 128, 1097, 1096, [1096, 458, 8], True, 978, 0),
    (5, 18, 48, 48, 64, 554, 549, [549, 446, 54, 274, 14], False, 0, 0),
    (5, 45, 16, 16, 64, 1063, 1059, [1059, 189, 657, 656, 32], True, 997, 0),
    (3, 9, 200, 100, 128, 445, 440, [440, 120, 3], False, 0, 0),
    (2, 3, 448, 64, 128, 1178, 1171, [1171, 2], True, 1148, 0),
    (2, 22, 1, 1, 64, 142, 141, [141, 13], True, 35, 0),
    (2, 36, 1, 1, 64, 322, 313, [313, 16], True, 213, 0),
    (3, 18, 48, 48, 64, 973, 973, [973, 372, 14], True, 885, 37),
    (4, 9, 64, 32, 64, 1106, 1106, [1106, 312, 269, 8], True, 1020, 3),
    (4, 10, 200, 100, 128, 420, 414, [414, 169, 247, 6], True, 398, 0),
    (3, 12, 192, 48, 128, 919, 918, [918, 193, 1], True, 790, 70),
    (3, 67, 32, 32, 128, 1677, 1677, [1677, 709, 43], True, 1607, 0),
    (3, 134, 16, 16, 128, 1777, 1776, [1776, 365, 122], True, 1575, 5),
    (3, 134, 16, 16, 128, 1676, 1668, [1668, 630, 42], False, 0, 0),
]

PLANTED = [
    # long lists in many runs: two column tiles, one, and the kernels of many rows
    (2, 3, 16, 2, 64, 33100, 33000, [33000, 20001], True, 0, 0),
    (1, 8, 6, 2, 128, 65700, 65667, None, True, 0, 0),
    (2, 8, 6, 2, 128, 66100, 66000, [66000, 40000], True, 33000, 70),
    (2, 5, 8, 2, 64, 66100, 66000, [65999, 33090], True, 33000, 3),
    (1, 1, 32, 8, 128, 32800, 32753, None, True, 0, 0),
    (1, 4, 4, 1, 64, 20000, 20000, None, False, 0, 0),
    (1, 1, 4, 2, 128, 30000, 30000, None, True, 20000, 100),
    (3, 3, 4, 1, 64, 9000, 9000, [9000, 5001, 2], True, 4000, 4),
    (3, 2, 71, 1, 64, 5000, 5000, [5000, 3001, 64], True, 1024, 4),
    (1, 40, 4, 2, 128, 9000, 9000, None, True, 5000, 5),
    (1, 40, 4, 2, 64, 9000, 9000, None, True, 5000, 5),
    (2, 100, 8, 8, 64, 3000, 2990, [2990, 1500], True, 0, 0),
    (3, 133, 16, 16, 128, 1672, 1672, [1672, 1500, 130], True, 0, 0),
    (1, 150, 24, 12, 128, 600, 600, None, True, 0, 0),
    (1, 150, 24, 12, 64, 600, 600, None, True, 90, 5),
    (2, 40, 8, 4, 128, 700, 700, [700, 30], True, 300, 37),
]


def masks(B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks):
    """What a case's masks do: `window`: some sequence has keys in front of every window, `sinks`: some of them are seen."""
    n = [kv_len] * B if lens is None else lens
    gap = window > 0 and any(x - S - window + 1 > sinks for x in n)
    padding = any(0 < x < S for x in n)
    res = {"sinks" if sinks else "window"} if gap else set()
    res |= {"padding"} if padding else set()
    res |= {"window+padding"} if gap and padding else set()
    res |= set() if causal else {"all keys"}
    res |= {"all keys+padding"} if padding and not causal else set()
    return res


def _places(n, S, window, sinks, tile, runs):
    """Keys where a kernel's work may be cut: the ends of the list, of the sinks and of the first and last token's window, and the
    borders of tiles and runs of the list of all S tokens."""
    first = max(n - S, 0)
    lo = max(0, first - window + 1) if window else 0
    gap = lo - sinks if lo > sinks else 0
    key = lambda l: l + (gap if gap and l >= sinks else 0)
    tiles = (n - gap + tile - 1) // tile
    per = (tiles + runs - 1) // runs
    at = {0, 1, n - 2, n - 1, sinks - 1, sinks, first, first + 1}
    for pos in (first, n - 1) if window else ():
        at |= {pos - window, pos - window + 1}
    for r in range(0, tiles, per):
        at |= {key(r * tile - 1), key(r * tile)}
    for r in list(range(1, min(9, tiles))) + list(range(max(tiles - 9, 1), tiles)):  # (tiles are of 32 keys, or of two halves)
        at |= {key(r * tile - 1), key(r * tile), key(r * tile + tile // 2 - 1), key(r * tile + tile // 2)}
    return sorted(x for x in at if 0 <= x < n)


def planted(case, dtype, four_bit, tile, runs):
    """Caches in which a few keys have nearly all the weight, as much each, and the others' values are zero: a planted key's value is
    one in a channel that it shares with two or three others, so that one key that is missing, or counted twice, shows.
    -> q, (k_cache, v_cache, k_scales, v_scales), k and v in fp64, lengths, planted keys of each sequence"""
    B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks = case
    n = [kv_len] * B if lens is None else lens
    g = torch.Generator().manual_seed(S + kv_len)
    k = 0.1 * torch.randn(B, Hkv, rows, D, generator=g)
    v = torch.zeros(B, Hkv, rows, D)
    at = [_places(x, S, window, sinks, tile, runs) for x in n]
    for b in range(B):
        for hk in range(Hkv):
            k[b, hk, at[b]] = 2.0
            for j, key in enumerate(at[b]):
                v[b, hk, key, (j + 5 * hk + 11 * b) % D] = 1.0
    k, v = k.to(dtype), v.to(dtype)
    q = torch.ones(B * S, Hq * D, dtype=dtype)
    if not four_bit:
        return q, (k, v, None, None), k.double(), v.double(), n, at
    (kc, kx), (vc, vx) = oc.fp4_encode(k), oc.fp4_encode(v)
    return q, (kc, vc, kx, vx), oc.fp4_decode(kc, kx), oc.fp4_decode(vc, vx), n, at


def planted_tolerance(D, n, dtype, mag, out):
    """cache_util.attention_tolerance without its term for probabilities below fp16's normal range: those have the value zero here,
    the others are one at least before the division.  A score is D products of 1 and 2, scaled: 2 * sqrt(D)."""
    e_s = (D + 16) * 2.0 ** -24 * 2.0 * math.sqrt(D)
    e_l = (max(n) / 16 + 64) * 2.0 ** -24
    return (UNIT[dtype] * (mag + out.abs()) + (2 * e_s + 2 * e_l) * mag) * 1.01 + 2.0 ** -24, e_s + e_l
