"""Calls of blocks.CachedAttention beside one another and with values that are no numbers, on the GPU."""
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
