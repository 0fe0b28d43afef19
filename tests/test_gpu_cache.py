"""GPU parity of the caches of several sequences (tri_cache_append, tri_cache_read, tri_cache_attention) with oracle/cache.py,
which computes in fp64.  4-bit codes and what is read back are compared exactly, attention within the bound that its
roundings give (cache_util.attention_tolerance).  Rows of the caches that a call has no business with hold NaN."""
import math

import pytest
import torch

import oracle
from cache_util import assert_within, attention_tolerance, make_caches, values
from oracle import cache as oc
from trinity_amd import blocks, ext
from util import assert_close, attn_inputs

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _lens(lens, dev):
    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)


def _poison(cache, scales, b, hk, keys):
    """Rows that nothing may read: NaN in either format."""
    if scales is None:
        cache[b, hk, keys] = math.nan
    else:
        scales[b, hk, keys] = 255


def _same(got, want):
    """The same values; NaN, what a block with an infinity or NaN reads as, is one of them."""
    none = torch.isnan(want)
    return torch.equal(torch.isnan(got), none) and torch.equal(got.masked_fill(none, 0), want.masked_fill(none, 0))


# ---------------------------------------------------------------------------------------------------- writing and reading
ROWS = [
    # B, S, Hkv, D, rows, kv_len, lens
    (1, 1, 8, 128, 40, 33, None),
    (3, 7, 2, 64, 20, 20, [20, 3, 0]),
    (2, 100, 3, 128, 130, 129, [129, 57]),
    (4, 1, 1, 64, 1, 1, [1, 0, 1, 1]),
    (2, 33, 1, 128, 50, 40, [1000000, -7]),  # lengths outside [0, kv_len] count as the nearer end
    (70, 2, 3, 64, 5, 5, None),
    (3, 700, 4, 128, 702, 701, [701, 333, 0]),  # so many rows that threads take several
    (2, 2100, 4, 64, 2100, 2100, [2100, 2099]),
]


@pytest.mark.parametrize("B,S,Hkv,D,rows,kv_len,lens", ROWS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("four_bit", [True, False])
@pytest.mark.parametrize("layout", ["bhld", "blhd"])
def test_append_and_read(dev, B, S, Hkv, D, rows, kv_len, lens, dtype, four_bit, layout):
    g = torch.Generator().manual_seed(B * 1000 + S)
    qkv = torch.randn(B * S, 3 * Hkv * D, generator=g)
    qkv[:, Hkv * D:2 * Hkv * D] *= torch.exp(3 * torch.randn(Hkv * D, generator=g))
    qkv = qkv.to(dtype)
    k, v = qkv[:, Hkv * D:2 * Hkv * D], qkv[:, 2 * Hkv * D:]
    caches = make_caches(7, B, Hkv, rows, D, dtype, four_bit, layout)
    d = [None if c is None else c.to(dev) for c in caches]
    if layout == "blhd" and Hkv > 1:
        assert d[0].stride(1) == d[0].shape[3]
    ld, dq = _lens(lens, dev), qkv.to(dev)
    op = blocks.CachedAttention(Hkv, Hkv, D)
    op.append(dq[:, Hkv * D:2 * Hkv * D], dq[:, 2 * Hkv * D:], d[0], d[1], d[2], d[3], lens=ld, kv_len=kv_len)
    n = [kv_len if lens is None else min(max(x, 0), kv_len) for x in (lens or [0] * B)]
    for x, cache, scales, got, gots in ((k, caches[0], caches[2], d[0], d[2]), (v, caches[1], caches[3], d[1], d[3])):
        want, wants = cache.clone(), None if scales is None else scales.clone()
        new = x.reshape(B, S, Hkv, D).transpose(1, 2)
        for b in range(B):
            m = min(S, n[b])
            if four_bit:
                want[b, :, n[b] - m:n[b]], wants[b, :, n[b] - m:n[b]] = oc.fp4_encode(new[b, :, S - m:])
            else:
                want[b, :, n[b] - m:n[b]] = new[b, :, S - m:]
        assert torch.equal(got.cpu(), want)
        assert wants is None or torch.equal(gots.cpu(), wants)
    # ... and back, in both types: more rows than the shorter sequences have
    for out_type in (F16, BF16) if four_bit else (dtype,):
        for many in (S, kv_len):
            rk, rv = op.read(d[0], d[1], d[2], d[3], dtype=out_type, rows=many, lens=ld, kv_len=kv_len)
            for got, cache, scales in ((rk, d[0], d[2]), (rv, d[1], d[3])):
                val = values(cache.cpu(), None if scales is None else scales.cpu())
                want = torch.zeros(B, Hkv, many, D, dtype=torch.float64)
                for b in range(B):
                    m = min(many, n[b])
                    want[b, :, many - m:] = val[b, :, n[b] - m:n[b]]
                assert _same(got.cpu(), want.to(out_type))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_of_every_value(dev, dtype):
    """All 65536 bit patterns: among like magnitudes and among unlike ones, infinities and NaN in some blocks."""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    for rows in (x.view(-1, 128), x.view(128, -1).t().contiguous()):
        n = rows.shape[0]
        codes, scales = blocks.CachedAttention.make_cache(1, 1, n, 128, dev)
        c2, s2 = codes.clone(), scales.clone()
        op = blocks.CachedAttention(1, 1, 128)
        op.append(rows.to(dev), rows.flip(0).to(dev), codes, c2, scales, s2)
        want, wants = oc.fp4_encode(rows)
        assert torch.equal(scales.cpu()[0, 0], wants) and torch.equal(codes.cpu()[0, 0], want)
        assert torch.equal(c2.cpu()[0, 0].flip(0), want)
        got = op.read(codes, c2, scales, s2, dtype=dtype)[0][0, 0].cpu()
        val = oc.fp4_decode(want, wants)
        assert _same(got, val.to(dtype))


# ------------------------------------------------------------------------------------------------------------- attention
ATTN = [
    # B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks
    (1, 1, 8, 2, 128, 1, 1, None, True, 0, 0),
    (1, 1, 32, 8, 128, 1100, 1025, None, True, 0, 0),
    (3, 1, 4, 4, 64, 300, 300, [300, 1, 0], True, 0, 0),
    (2, 1, 71, 1, 64, 700, 700, [699, 64], True, 0, 0),
    (5, 2, 8, 1, 128, 520, 515, [515, 1, 2, 65, 0], True, 0, 0),
    (1, 5, 4, 2, 64, 70, 65, None, False, 0, 0),
    (2, 40, 6, 3, 128, 200, 190, [190, 17], False, 0, 0),
    (1, 130, 4, 1, 64, 130, 130, None, True, 0, 0),
    (2, 257, 2, 2, 128, 300, 300, [300, 100], True, 0, 0),
    (1, 64, 9, 3, 128, 2000, 2000, None, True, 0, 0),
    (1, 33, 71, 1, 64, 400, 400, None, True, 0, 0),
    (1, 1, 4, 1, 128, 600, 600, None, True, 100, 4),
    (3, 1, 8, 2, 64, 900, 900, [900, 130, 5], True, 64, 70),   # as many sinks as keys, or nearly
    (2, 3, 71, 1, 64, 640, 640, [640, 200], True, 128, 4),
    (1, 300, 4, 2, 128, 300, 300, None, True, 17, 3),
    (2, 100, 8, 2, 128, 500, 500, [500, 60], True, 33, 0),
    (1, 200, 2, 1, 64, 700, 700, None, True, 1, 1),            # a token and the first one
    (1, 4, 4, 4, 128, 260, 260, None, True, 1000, 8),           # a window wider than the sequence
    (4, 16, 4, 2, 128, 128, 100, [100, 99, 16, 15], True, 64, 64),
    (1, 128, 32, 8, 128, 640, 640, None, True, 256, 4),
    (12, 1, 16, 2, 128, 400, 400, [400 - 31 * i for i in range(12)], True, 0, 0),
    (1, 7, 12, 2, 64, 3000, 2900, None, True, 0, 0),
    (1, 8, 8, 2, 128, 5000, 5000, None, False, 0, 0),
    (1, 512, 4, 1, 64, 1500, 1500, None, True, 0, 0),
    (1, 1, 8, 2, 128, 640, 640, None, True, 0, 0),             # few rows: one run in 4 bits, several in 16
    (33, 1, 4, 4, 64, 1300, 1300, [1300 - 40 * i for i in range(33)], True, 0, 0),  # many heads: 1024 keys and fewer in one run
    (33, 1, 4, 4, 64, 900, 900, [900 - 27 * i for i in range(33)], True, 0, 0),
    (1, 8, 16, 4, 64, 2000, 1990, None, True, 0, 0),
    (2, 8, 16, 4, 64, 200, 200, [200, 91], True, 60, 4),
    (1, 8, 16, 4, 128, 200, 200, None, True, 0, 0),
    # column tiles of 16 rows, two of them (4 bits, many keys of all KV heads together), in one run and in several
    (43, 8, 18, 6, 64, 520, 513, [513 - 11 * i for i in range(43)], True, 0, 0),
    (33, 5, 32, 8, 128, 500, 498, [498 - 15 * i for i in range(33)], True, 0, 0),
    (2, 3, 16, 2, 64, 33100, 33000, [33000, 20001], True, 0, 0),
    (1, 8, 6, 2, 128, 65700, 65667, None, True, 0, 0),
    # two key ways: in one run and in several
    (1, 48, 48, 48, 64, 329, 329, None, True, 0, 0),
    (2, 155, 8, 8, 64, 340, 339, [339, 150], True, 200, 3),
    (3, 48, 32, 32, 64, 660, 653, [653, 640, 20], True, 0, 0),
    (3, 20, 96, 48, 128, 840, 840, [840, 100, 19], True, 0, 0),
    (3, 133, 16, 16, 128, 1672, 1672, [1672, 1500, 130], False, 0, 0),
    (1, 100, 71, 1, 64, 1500, 1500, None, True, 0, 0),
    (2, 66, 71, 1, 64, 420, 411, [411, 350], True, 97, 33),    # lists that end in either half of a tile, sinks into the second
    (3, 129, 2, 1, 64, 290, 289, [289, 161, 130], True, 0, 0),
]


def _case(dev, B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks, dtype, four_bit, layout="bhld", seed=1, scratch=None):
    caches = make_caches(seed, B, Hkv, rows, D, dtype, four_bit, layout)
    n = [kv_len] * B if lens is None else lens
    for b in range(B):
        seen = oc.visible(n[b], S, causal, window, sinks).any(0)
        dead = torch.cat((~seen, torch.ones(rows - n[b], dtype=torch.bool)))
        for cache, scales in ((caches[0], caches[2]), (caches[1], caches[3])):
            _poison(cache, scales, b, slice(None), dead)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(B * S, Hq * D, generator=g).to(dtype)
    k, v = values(caches[0], caches[2]), values(caches[1], caches[3])
    want, lse, mag = oc.cache_attention(q, k, v, n, n_q_heads=Hq, causal=causal, window=window, sinks=sinks)
    tol, tol_lse = attention_tolerance(q, k, v, n, mag, want, dtype, n_q_heads=Hq, scale=D ** -0.5)
    d = [None if c is None else c.to(dev) for c in caches]
    return q.to(dev), d, _lens(lens, dev), want, lse, tol, tol_lse


def _check(got, got_lse, want, lse, tol, tol_lse):
    assert_within(got, want, tol, "out")
    if got_lse is not None:
        got_lse = got_lse.cpu().double()
        none = lse == -math.inf
        assert torch.equal(got_lse == -math.inf, none)
        assert_within(got_lse.masked_fill(none, 0), lse.masked_fill(none, 0), tol_lse + 2.0 ** -21 + lse.abs().masked_fill(none, 0) * 2.0 ** -22, "lse")


@pytest.mark.parametrize("B,S,Hq,Hkv,D,rows,kv_len,lens,causal,window,sinks", ATTN)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("four_bit", [False, True])
def test_attention(dev, B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks, dtype, four_bit):
    q, c, ln, *ref = _case(dev, B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks, dtype, four_bit)
    op = blocks.CachedAttention(Hq, Hkv, D, causal=causal, window=window, sinks=sinks)
    out = torch.full((B * S, Hq * D), math.nan, dtype=dtype, device=dev)
    got, lse = op.attend(q, c[0], c[1], c[2], c[3], lens=ln, kv_len=kv_len, out=out, want_lse=True)
    assert got is out
    _check(got, lse, *ref)
    # without the log-sum-exp the same bits
    assert torch.equal(op.attend(q, c[0], c[1], c[2], c[3], lens=ln, kv_len=kv_len), out)


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("i", [1, 3, 8, 9, 13, 15, 21])
def test_attention_strides_and_scratch(dev, i, four_bit):
    """Heads of a position next to one another, q among other columns, a wide output; less scratch than asked for."""
    B, S, Hq, Hkv, D, rows, kv_len, lens, causal, window, sinks = ATTN[i]
    q, c, ln, *ref = _case(dev, *ATTN[i], F16, four_bit, "blhd", seed=9)
    p = ext.cache_params(B, Hkv, D, S, kv_len, n_q_heads=Hq, causal=causal, window=window, sinks=sinks)
    need = ext.cache_scratch_bytes(p, four_bit)
    wide_q = torch.full((B * S, Hq * D + 24), math.nan, dtype=F16, device=dev)
    wide_q[:, 16:16 + Hq * D] = q
    for bytes_ in {0, need // 3, need // 2, need}:
        wide_o = torch.full((B * S, Hq * D + 8), 7.0, dtype=F16, device=dev)
        scratch = torch.full((bytes_,), 255, dtype=torch.uint8, device=dev) if bytes_ else None
        lse = torch.full((B, Hq, S), math.nan, device=dev)
        ext.cache_attention(wide_q[:, 16:16 + Hq * D], c[0], c[2], c[1], c[3], ln, scratch, lse, wide_o[:, :Hq * D], p)
        _check(wide_o[:, :Hq * D], lse, *ref)
        assert bool((wide_o[:, Hq * D:] == 7).all())


def test_one_sequence_without_a_batch_dimension(dev):
    q, c, ln, *ref = _case(dev, 1, 3, 4, 2, 64, 90, 80, None, True, 16, 2, BF16, True)
    op = blocks.CachedAttention(4, 2, 64, window=16, sinks=2)
    got = op.attend(q, c[0][0], c[1][0], c[2][0], c[3][0], kv_len=80)
    assert_within(got, ref[0], ref[2], "out")


def test_large_scores_and_lazy_maximum(dev):
    """Scores that climb by hundreds along the keys, and a single key far above the others."""
    B, S, Hq, Hkv, D, n = 1, 2, 4, 2, 128, 700
    for four_bit in (False, True):
        q, c, ln, *_ = _case(dev, B, S, Hq, Hkv, D, n, n, None, True, 0, 0, F16, False, seed=5)
        k = c[0].cpu()
        k[:] = k * (torch.arange(n)[None, None, :, None] / n).half() * 3
        k[:, :, 333] = 6.0 * torch.sign(q.cpu().view(1, S, Hq, D)[:, 0, ::2].unsqueeze(2)[:, :, 0])
        caches = (k, c[1].cpu(), None, None)
        if four_bit:
            (kc, kx), (vc, vx) = oc.fp4_encode(k), oc.fp4_encode(caches[1])
            caches = (kc, vc, kx, vx)
        kv, vv = values(caches[0], caches[2]), values(caches[1], caches[3])
        want, lse, mag = oc.cache_attention(q, kv, vv, [n], n_q_heads=Hq)
        tol, tol_lse = attention_tolerance(q, kv, vv, [n], mag, want, F16, n_q_heads=Hq, scale=D ** -0.5)
        op = blocks.CachedAttention(Hq, Hkv, D)
        got = op.attend(q, *[None if x is None else x.to(dev) for x in caches], want_lse=True)
        _check(got[0], got[1], want, lse, tol, tol_lse)


def test_numbers_that_are_none_stay_where_they_are_seen(dev):
    """A NaN or infinity in a key or value reaches the tokens that see it, and no other sequence or KV head."""
    B, S, Hq, Hkv, D, n = 3, 1, 4, 2, 128, 500
    for four_bit in (False, True):
        q, c, ln, want, lse, tol, tol_lse = _case(dev, B, S, Hq, Hkv, D, n, n, None, True, 0, 0, F16, four_bit)
        for i in (0, 1):  # key 450 of (1, 0) in K, of (1, 1) in V
            if four_bit:
                c[2 + i][1, i, 450] = 255
            else:
                c[i][1, i, 450, 3] = math.nan
        got = blocks.CachedAttention(Hq, Hkv, D).attend(q, c[0], c[1], c[2], c[3]).cpu().view(B, Hq, D)
        assert torch.isnan(got[1, :2]).all() and torch.isnan(got[1, 2:, 3]).all()
        others = got[[0, 2]].reshape(2, -1)
        assert_within(others, want.view(B, -1)[[0, 2]], tol.view(B, -1)[[0, 2]], "other sequences")


@pytest.mark.parametrize("S,Hq,D", [(1, 4, 128), (9, 2, 64), (40, 4, 128), (70, 2, 64)])
@pytest.mark.parametrize("four_bit", [False, True])
def test_runs_that_see_no_number(dev, S, Hq, D, four_bit):
    """Parts of the keys whose scores are NaN one and all, and a query that is one, are not lost in the merge of the parts."""
    Hkv, n = 1, 4096
    q, c, ln, want, lse, tol, tol_lse = _case(dev, 1, S, Hq, Hkv, D, n, n, None, False, 0, 0, BF16, four_bit)
    assert ext.cache_scratch_bytes(ext.cache_params(1, Hkv, D, S, n, n_q_heads=Hq, causal=False), four_bit) > 0
    op = blocks.CachedAttention(Hq, Hkv, D, causal=False)
    row = (S // 2, Hq - 1)  # token, head
    bad = q.clone().view(S, Hq, D)
    bad[row] = math.nan
    got, got_lse = op.attend(bad.view(S, -1), *c, want_lse=True)
    got, got_lse = got.cpu().view(S, Hq, D), got_lse.cpu()[0]
    assert torch.isnan(got[row]).all() and torch.isnan(got_lse[row[1], row[0]])
    rest = torch.ones(S, Hq, dtype=torch.bool)
    rest[row] = False
    assert_within(got[rest], want.view(S, Hq, D)[rest], tol.view(S, Hq, D)[rest], "other rows")
    (c[2] if four_bit else c[0])[:, :, 1024:2560] = 255 if four_bit else math.nan  # K of whole parts
    got, got_lse = op.attend(q, *c, want_lse=True)
    assert torch.isnan(got).all() and torch.isnan(got_lse).all()


@pytest.mark.parametrize("four_bit", [False, True])
def test_offsets_beyond_32_bits(dev, four_bit):
    """A cache whose rows lie so far apart that their offsets do not fit 32 bits (in elements, and in bytes)."""
    n, D, Hkv = 2100, 64, 2
    step = 1 << (21 if four_bit else 20)
    caches = make_caches(3, 1, Hkv, n, D, BF16, four_bit)
    far = []
    for cache in caches[:2]:
        flat = torch.empty(n * step + (1 << 12), dtype=cache.dtype, device=dev)
        view = flat.as_strided((1, Hkv, n, cache.shape[3]), (0, 256, step, 1))
        view.copy_(cache.to(dev))
        far.append(view)
    scales = [None if s is None else s.to(dev) for s in caches[2:]]
    g = torch.Generator().manual_seed(2)
    q = torch.randn(3, 4 * D, generator=g).to(BF16)
    k, v = values(caches[0], caches[2]), values(caches[1], caches[3])
    for window, sinks in ((0, 0), (100, 5)):
        want, lse, mag = oc.cache_attention(q, k, v, [n], n_q_heads=4, window=window, sinks=sinks)
        tol, tol_lse = attention_tolerance(q, k, v, [n], mag, want, BF16, n_q_heads=4, scale=D ** -0.5)
        op = blocks.CachedAttention(4, Hkv, D, window=window, sinks=sinks)
        got = op.attend(q.to(dev), *far, *scales, want_lse=True)
        _check(*got, want, lse, tol, tol_lse)
    rk, rv = op.read(*far, *scales, dtype=BF16, rows=50)
    assert torch.equal(rk.cpu().double(), k[:, :, n - 50:]) and torch.equal(rv.cpu().double(), v[:, :, n - 50:])
    new = torch.randn(1, Hkv * D, generator=g).to(BF16)
    op.append(new.to(dev), new.to(dev), *far, *scales)
    back = op.read(*far, *scales, dtype=BF16, rows=1)[0].cpu().view(1, -1)
    assert torch.equal(back, oc.fp4_decode(*oc.fp4_encode(new)).to(BF16) if four_bit else new)


# ----------------------------------------------------------------------------------------------------- used together
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_prompt_then_tokens(dev, four_bit, window, sinks):
    """Two conversations: prompts of different lengths in one padded call, then single tokens, each written and attended to;
    every step against the oracle on what the cache holds by then."""
    B, Hq, Hkv, D, rows, dtype = 2, 8, 2, 128, 160, F16
    lens = [90, 51]
    g = torch.Generator().manual_seed(11)
    op = blocks.CachedAttention(Hq, Hkv, D, window=window, sinks=sinks)
    if four_bit:
        (kc, kx), (vc, vx) = (op.make_cache(B, Hkv, rows, D, dev) for _ in range(2))
    else:
        kc, vc = (torch.full((B, Hkv, rows, D), math.nan, dtype=dtype, device=dev) for _ in range(2))
        kx = vx = None
    hist = torch.zeros(2, B, Hkv, rows, D, dtype=torch.float64)
    steps = [max(lens)] + [1] * 5
    n = list(lens)
    for step, S in enumerate(steps):
        if step:
            n = [x + 1 for x in n]
        q, k, v = (torch.randn(B * S, h * D, generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
        ln = _lens(n, dev)
        op.append(k.to(dev), v.to(dev), kc, vc, kx, vx, lens=ln)
        got, lse = op.attend(q.to(dev), kc, vc, kx, vx, lens=ln, want_lse=True)
        for i, x in enumerate((k, v)):
            val = oc.fp4_decode(*oc.fp4_encode(x)) if four_bit else x.double()
            val = val.view(B, S, Hkv, D).transpose(1, 2)
            for b in range(B):
                m = min(S, n[b])
                hist[i, b, :, n[b] - m:n[b]] = val[b, :, S - m:]
        want, wlse, mag = oc.cache_attention(q, hist[0], hist[1], n, n_q_heads=Hq, window=window, sinks=sinks)
        tol, tol_lse = attention_tolerance(q, hist[0], hist[1], n, mag, want, dtype, n_q_heads=Hq, scale=D ** -0.5)
        _check(got, lse, want, wlse, tol, tol_lse)


@pytest.mark.parametrize("S,P,prenorm,qknorm", [(48, 0, False, False), (1, 300, True, False), (7, 90, True, True), (130, 60, False, True)])
def test_plan_is_the_block(dev, S, P, prenorm, qknorm):
    """One sequence, 16-bit, no window: the block of tri_qkv_attention (blocks.AttentionPlan) and its oracle.  The plans
    round the same values (q, k, v, the normalised x) to 16 bits and differ in the order of their sums: 1e-2 as for the block."""
    N, Hq, Hkv, D = 256, 4, 2, 128
    t = attn_inputs(S, N, Hq, Hkv, D, P=P, w_std=0.06, with_cache=True)
    want = oracle.qkv_attention(t["x"], t["wq"], t["wk"], t["wv"], n_q_heads=Hq, n_kv_heads=Hkv, head_dim=D, scale=D ** -0.5,
                                causal=True, kv_prefix=P, k_cache=t["k_cache"], v_cache=t["v_cache"], prenorm=prenorm,
                                prenorm_weight=t["norm_w"] if prenorm else None, qknorm=qknorm, rms_eps=1e-5, want_lse=True)
    d = {k: v.to(dev) for k, v in t.items()}
    kc, vc = d["k_cache"].clone()[None], d["v_cache"].clone()[None]
    plan = blocks.CachedAttentionPlan(Hq, Hkv, D, prenorm=prenorm, qknorm=qknorm, eps=1e-5)
    out = torch.full((S, Hq * D), math.nan, dtype=F16, device=dev)
    got, lse = plan.run(d["x"], d["wq"], d["wk"], d["wv"], out, kc, vc, kv_len=P + S, norm_w=d["norm_w"] if prenorm else None,
                        want_lse=True)
    assert got is out
    assert_close(out, want["O2"], 1e-2, 1e-2, "O2")
    assert_close(lse[0], want["lse"], 1e-2, 1e-2, "lse")
    assert_close(kc[0, :, P:P + S], want["k_new"], 1e-2, 1e-2, "appended k")
    assert_close(vc[0, :, P:P + S], want["v_new"], 1e-2, 1e-2, "appended v")
    assert torch.equal(kc[0, :, :P], d["k_cache"][:, :P])
    other = torch.empty_like(out)
    blocks.AttentionPlan("vanilla", D=D, H=Hq, P=P, prenorm=prenorm, qknorm=qknorm, scale=D ** -0.5, causal=True, n_kv_heads=Hkv,
                         eps=1e-5).run(d["x"], d["wq"], d["wk"], d["wv"], other, d["k_cache"], d["v_cache"],
                                       norm_w=d["norm_w"] if prenorm else None)
    assert_close(out, other.cpu(), 1e-2, 1e-2, "the two blocks")


def test_plan_over_ragged_four_bit_caches(dev):
    """The block for three conversations, padded, in bf16 and a window: its attention is that over the cache it leaves behind."""
    B, S, N, Hq, Hkv, D, rows = 3, 40, 192, 6, 2, 64, 90
    lens = [90, 33, 5]
    t = attn_inputs(B * S, N, Hq, Hkv, D, w_std=0.07)
    t = {k: v.to(BF16) for k, v in t.items()}
    d = {k: v.to(dev) for k, v in t.items()}
    plan = blocks.CachedAttentionPlan(Hq, Hkv, D, window=25, sinks=2)
    (kc, kx), (vc, vx) = (plan.attention.make_cache(B, Hkv, rows, D, dev) for _ in range(2))
    before = make_caches(4, 1, Hkv, 50, D, BF16, True)
    for new, old in zip((kc, vc, kx, vx), before):
        new[0, :, :50] = old[0].to(dev)
    out = plan.run(d["x"], d["wq"], d["wk"], d["wv"], torch.empty(B * S, Hq * D, dtype=BF16, device=dev), kc, vc, kx, vx,
                   lens=_lens(lens, dev))
    k, v = values(kc.cpu(), kx.cpu()), values(vc.cpu(), vx.cpu())
    assert torch.equal(kc[0, :, :50].cpu(), before[0][0])
    # the rows written: of k = x.wk in 16 bits, within a step of 4 bits of the exact product (its rounding may move a code)
    exact = (t["x"].double() @ t["wk"].double()).view(B, S, Hkv, D).transpose(1, 2)
    for b, n in enumerate(lens):
        m = min(S, n)
        unit = torch.ldexp(torch.ones(Hkv, m, D // 32, dtype=torch.float64), kx[b, :, n - m:n].cpu().long() - 127).repeat_interleave(32, -1)
        assert bool(((k[b, :, n - m:n] - exact[b, :, S - m:]).abs() <= 1.1 * unit).all())
    q = (t["x"].float() @ t["wq"].float()).to(BF16)
    want, lse, mag = oc.cache_attention(q, k, v, lens, n_q_heads=Hq, window=25, sinks=2)
    assert_close(out, want, 2e-2, 2e-2, "out")


@pytest.mark.parametrize("four_bit", [False, True])
def test_graph_of_a_decode_step(dev, four_bit):
    """A step captured once, on a stream of its own, and replayed as the lengths grow on the device; eager calls of the same
    objects and of another shape between the replays, on the graph's stream too; two graphs of one object."""
    B, Hq, Hkv, D, rows, dtype = 3, 16, 4, 128, 3000, F16
    caches = make_caches(5, B, Hkv, rows, D, dtype, four_bit)
    c = [None if x is None else x.to(dev) for x in caches]
    start = [2900, 700, 0]
    g = torch.Generator().manual_seed(6)
    op = blocks.CachedAttention(Hq, Hkv, D)
    win = blocks.CachedAttention(Hq, Hkv, D, window=2500, sinks=4)
    lens = _lens(start, dev)
    q, k, v = (torch.zeros(B, h * D, dtype=dtype, device=dev) for h in (Hq, Hkv, Hkv))
    out, out2 = (torch.zeros(B, Hq * D, dtype=dtype, device=dev) for _ in range(2))
    kv = dict(lens=lens, kv_len=rows)

    def step(o, dst):
        lens.add_(1)
        op.append(k, v, c[0], c[1], c[2], c[3], **kv)
        o.attend(q, c[0], c[1], c[2], c[3], out=dst, **kv)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(op, out)
        step(win, out2)
    stream.synchronize()
    kept = {id(o): dict(o._scratch) for o in (op, win)}
    assert all(len(x) == 1 for x in kept.values())
    lens.copy_(torch.tensor(start))
    for x, y in zip(c, caches):
        if x is not None:
            x.copy_(y)
    graphs = []
    for o, dst in ((op, out), (win, out2)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(o, dst)
        graphs.append(graph)
    assert all(dict(o._scratch) == kept[id(o)] for o in (op, win))  # the graphs have scratch of their own
    n = list(start)
    hist = [values(caches[0], caches[2]).clone(), values(caches[1], caches[3]).clone()]
    for rep in range(6):
        new = [torch.randn(B, h * D, generator=g).to(dtype) for h in (Hq, Hkv, Hkv)]
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        torch.cuda.synchronize()
        which = rep % 2
        with torch.cuda.stream(stream):
            graphs[which].replay()
        stream.synchronize()
        n = [x + 1 for x in n]
        for i in (0, 1):
            val = oc.fp4_decode(*oc.fp4_encode(new[1 + i])) if four_bit else new[1 + i].double()
            for b in range(B):
                hist[i][b, :, n[b] - 1] = val.view(B, Hkv, D)[b]
        kw = dict(window=2500, sinks=4) if which else {}
        want, lse, mag = oc.cache_attention(new[0], hist[0], hist[1], n, n_q_heads=Hq, **kw)
        tol, _ = attention_tolerance(new[0], hist[0], hist[1], n, mag, want, dtype, n_q_heads=Hq, scale=D ** -0.5)
        got = (out, out2)[which]
        assert_within(got, want, tol, "replay %d" % rep)
        eager = (op, win)[which].attend(q, c[0], c[1], c[2], c[3], **kv)
        assert torch.equal(eager, got)
        with torch.cuda.stream(stream):
            for other in (op, win):
                other.attend(q[:1].repeat(B * 3, 1), c[0], c[1], c[2], c[3], **kv)
        torch.cuda.synchronize()


def test_plan_keeps_no_buffer_that_a_graph_uses(dev):
    """A captured step of single tokens is replayed after eager prompts of the same plan, whose memory others have filled since,
    and beside another stream's step."""
    B, N, Hq, Hkv, D, rows = 4, 256, 8, 2, 128, 600
    t = {k: v.to(dev) for k, v in attn_inputs(40 * B, N, Hq, Hkv, D, w_std=0.06).items()}
    w = (t["wq"], t["wk"], t["wv"])
    plan = blocks.CachedAttentionPlan(Hq, Hkv, D, prenorm=True, qknorm=True, eps=1e-5)
    caches = [x.to(dev) for x in make_caches(8, B, Hkv, rows, D, F16, False)[:2]]
    lens = _lens([600, 41, 300, 77], dev)
    out, want = torch.zeros(B, Hq * D, dtype=F16, device=dev), torch.zeros(B, Hq * D, dtype=F16, device=dev)
    x = t["x"][:B].clone()
    run = lambda x, out, c: plan.run(x, *w, out, *c, lens=lens)
    run(x, out, caches)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(x, out, caches)
    side = torch.cuda.Stream()
    for rep in range(5):
        x.copy_(t["x"][rep * B:(rep + 1) * B])
        c = [y.clone() for y in caches]
        prompt = torch.empty(40 * B, Hq * D, dtype=F16, device=dev)
        run(t["x"], prompt, [y.clone() for y in caches])
        fill = [torch.full((n,), 0x7E, dtype=torch.uint8, device=dev) for n in (B * N * 2, B * Hq * D * 2, B * Hkv * D * 2, 1 << 18, 1 << 21)]
        run(x, want, c)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = run(t["x"], torch.empty_like(prompt), [y.clone() for y in c])
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep
        assert all(torch.equal(y, z) for y, z in zip(c, caches))
        assert all(bool((f == 0x7E).all()) for f in fill)
        del beside


def test_two_streams_and_a_captured_first_call(dev):
    """One object on two streams at a time, and captured before it has ever run: every one of them with scratch of its own."""
    q, c, ln, *ref = _case(dev, 1, 1, 32, 8, 128, 4000, 4000, None, True, 0, 0, F16, True)
    op = blocks.CachedAttention(32, 8, 128)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        captured = op.attend(q, c[0], c[1], c[2], c[3])
    assert not op._scratch
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            if i % 3 == 2:
                graph.replay()
            else:
                outs.append(op.attend(q, c[0], c[1], c[2], c[3]))
    torch.cuda.synchronize()
    assert len(op._scratch) == 2
    _check(outs[0], None, *ref)
    assert all(torch.equal(x, outs[0]) for x in outs + [captured])


def test_under_inference_mode(dev):
    q, c, ln, *ref = _case(dev, 2, 3, 4, 2, 64, 90, 90, [90, 20], True, 0, 0, F16, True)
    op = blocks.CachedAttention(4, 2, 64)
    with torch.inference_mode():
        out, lse = op.attend(q, c[0], c[1], c[2], c[3], lens=ln, want_lse=True)
        k, v = op.read(c[0], c[1], c[2], c[3], lens=ln)
        _check(out.clone(), lse + 0, *ref)
        assert (k + v).shape == (2, 2, 90, 64) and k.clone().is_contiguous()
    k, v = op.read(c[0], c[1], c[2], c[3], lens=ln)
    k += 1  # the results are tensors like others, also in place
    assert _same(v, op.read(c[0], c[1], c[2], c[3], lens=ln)[1])


def test_other_devices_tensors_are_refused(dev):
    q, c, ln, *_ = _case(dev, 2, 1, 4, 2, 64, 64, 64, [64, 3], True, 0, 0, F16, True)
    op = blocks.CachedAttention(4, 2, 64)
    with pytest.raises(ValueError):
        op.attend(q, c[0], c[1], c[2], c[3], lens=ln.cpu())
    with pytest.raises(ValueError):
        op.attend(q, c[0], c[1], c[2].cpu(), c[3], lens=ln)


def test_nothing_to_do(dev):
    """No sequences, no tokens, no keys."""
    op = blocks.CachedAttention(4, 2, 64)
    q = torch.randn(2, 256, dtype=torch.float32, device=dev).half()
    empty = torch.empty(2, 2, 0, 64, dtype=F16, device=dev)
    out, lse = op.attend(q, empty, empty, want_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    cache = torch.zeros(2, 2, 8, 64, dtype=F16, device=dev)
    assert op.attend(q[:0], cache, cache).shape == (0, 256)
    assert op.read(empty, empty, rows=3)[0].shape == (2, 2, 3, 64)
    assert not op.read(empty, empty, rows=3)[1].any()
    op.append(q[:, :128], q[:, :128], empty, empty)
    op.append(q[:0, :128], q[:0, :128], cache, cache)
    assert not cache.any()
