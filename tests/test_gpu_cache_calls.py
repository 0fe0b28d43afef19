"""Calls of blocks.CachedAttention beside one another and with values that are no numbers, on the GPU."""
import math
import threading

import pytest
import torch

from cache_util import make_caches
from trinity_amd import blocks

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def test_threads_on_one_stream(dev):
    """Two threads, one object, the default stream: calls of two launches each, whose scratch is their own."""
    Hq, Hkv, D, n = 8, 2, 128, 4000
    c = [x.to(dev) for x in make_caches(5, 1, Hkv, n, D, F16, True)]
    g = torch.Generator().manual_seed(3)
    qs = [torch.randn(1, Hq * D, generator=g).to(F16).to(dev) for _ in range(2)]
    op = blocks.CachedAttention(Hq, Hkv, D)
    want = [op.attend(q, *c).clone() for q in qs]
    assert op._scratch and not torch.equal(*want)
    torch.cuda.synchronize()
    off = [0, 0]

    def call(i):
        outs = [op.attend(qs[i], *c) for _ in range(300)]
        off[i] = sum(not torch.equal(x, want[i]) for x in outs)

    threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert off == [0, 0] and len(op._scratch) == 1


PADDED = [
    # S, Hq, Hkv, kv_len, lens: at most 16 stacked rows and at most 32, in one run and several, and more
    (4, 4, 2, 100, [100, 2]),
    (4, 4, 2, 4000, [3999, 3]),
    (8, 6, 2, 33000, [1000, 5]),
    (8, 24, 8, 700, [700, 7]),
    (40, 4, 2, 64, [64, 23]),
    (100, 4, 2, 2000, [1900, 60]),
    (100, 8, 8, 330, [330, 50]),
    (140, 32, 32, 1000, [999, 130]),
    (300, 64, 64, 300, [300, 170]),
    (8, 384, 128, 520, [520, 5]),
]


@pytest.mark.parametrize("S,Hq,Hkv,kv_len,lens", PADDED)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_padding_is_zero_beside_values_that_are_no_numbers(dev, S, Hq, Hkv, kv_len, lens, D, four_bit, bad):
    """Rows of padding see nothing: zeros and -inf, whatever stands in the values that other tokens of their sequence see."""
    B = len(lens)
    c = [None if x is None else x.to(dev) for x in make_caches(6, B, Hkv, kv_len, D, F16, four_bit)]
    if four_bit:
        c[3][1, :, 1] = 255
    else:
        c[1][1, :, 1] = bad
    q = torch.randn(B * S, Hq * D, generator=torch.Generator().manual_seed(4)).to(F16).to(dev)
    op = blocks.CachedAttention(Hq, Hkv, D)
    lens_ = torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = op.attend(q, *c, lens=lens_, kv_len=kv_len, want_lse=True)
    out = out.view(B, S, Hq, D)
    pad = S - lens[1]
    assert not out[1, :pad].any() and bool((lse[1, :, :pad] == -math.inf).all())
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(lse[1, :, pad:]).all())
    assert not bool(torch.isfinite(out[1, pad + 1:]).any()), "tokens that see the value"


@pytest.mark.parametrize("S,Hq", [(1, 4), (3, 71)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_row_whose_scores_are_all_minus_infinity(dev, S, Hq, D):
    """It has keys, unlike padding, and none of their weights is a number."""
    k = torch.full((1, 1, S, D), -math.inf, dtype=F16, device=dev)
    v = torch.ones(1, 1, S, D, dtype=F16, device=dev)
    out, lse = blocks.CachedAttention(Hq, 1, D).attend(torch.ones(S, Hq * D, dtype=F16, device=dev), k, v, want_lse=True)
    assert bool(torch.isnan(out).all()) and bool((lse == -math.inf).all())
