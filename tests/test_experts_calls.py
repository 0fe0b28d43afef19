"""The calls of perf/more_operators.py, its listed cases and some thousand of the range that it draws from, against the entry points'
own checks, on the CPU: none is refused.  (Descriptors without memory: checks read no elements.)"""
import importlib.util
import os
import random
import re

import pytest
import torch

from test_experts_plans import experts_plan
from trinity_amd import blocks, ext

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cases():
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _like(dtype, *shape, i32=False):
    """A contiguous tensor's descriptor, at an address that nothing reads."""
    s = ext.TriTensor()
    s.ptr, s.ndim = 1 << 20, len(shape)
    s.dtype = ext.TRI_I32 if i32 else ext._DTYPES[dtype]
    step = 1
    for i in reversed(range(len(shape))):
        s.shape[i], s.stride[i] = shape[i], step
        step *= shape[i]
    return s


def _status(mod, c):
    u8, f32 = torch.uint8, torch.float32
    dt = mod.DTYPES[c["dtype"]]
    four = lambda *shape: (_like(u8, *shape[:-1], shape[-1] // 2), _like(u8, *shape[:-1], shape[-1] // 32))
    if c["kind"] == "quantize":
        x, q = _like(dt, c["rows"], c["k"]), four(c["rows"], c["k"])
        return [ext.fp4_quantize(x, *q, validate_only=True), ext.fp4_dequantize(*q, x, validate_only=True)]
    if c["kind"] == "product":
        m, k, n = c["rows"], c["k"], c["n"]
        x = four(m, k) if c["x4"] else (_like(dt, m, k), None)
        need = ext.fp4_workspace_bytes(m, k, n, c["x4"])
        return [ext.fp4_matmul(*x, *four(n, k), _like(u8, need) if need else None, _like(dt, m, n), validate_only=True)]
    if c["kind"] == "route":
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        op = blocks.Router(k, scores=c["scores"], groups=c["groups"], top_groups=c["top_groups"], group_top=c["group_top"],
                           renormalize=c["renormalize"], scale=c["scale"])
        return [ext.route(_like(dt, t, e), _like(f32, e) if c["bias"] else None, _like(None, t, k, i32=True), _like(f32, t, k), op._p,
                          validate_only=True)]
    e, k, n, f = mod.EXPERTS[c["config"]]
    t = c["tokens"]
    w = lambda rows, deep: four(e, rows, deep) if c["w4"] else (_like(dt, e, rows, deep), None)
    need = ext.experts_workspace_bytes(t, k, e, n, f)
    return [ext.experts_ffn(_like(dt, t, n), _like(None, t, k, i32=True), _like(f32, t, k), *w(f, n), *w(f, n), *w(n, f), _like(u8, need),
                            _like(dt, t, n), validate_only=True)]


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_no_case_is_refused(seed):
    mod, rng = _cases(), random.Random(seed)
    for c in mod.listed() + [mod.draw(rng) for _ in range(3000)]:
        assert not any(_status(mod, c)), c


@pytest.mark.parametrize("E,k,N,F", [(8, 2, 4096, 14336), (64, 6, 4096, 1792), (32, 4, 4544, 2272), (5, 1, 512, 96)])
def test_rows_of_tiles_go_by_whole_tiles(E, k, N, F):
    """Beyond few rows the tile of 4-bit experts changes where one or one and a half of its largest are full, and nowhere else."""
    for mean, bm in ((64, 256), (150, 256), (192, 256), (193, 256), (208, 256), (209, 256), (256, 256), (257, 128), (384, 128), (385, 256),
                     (2000, 256)):
        T = mean * E // k
        if -(-T * k // E) == mean:  # (the plan's mean, rounded up)
            assert experts_plan(T, k, E, N, F, True)[0] == bm, mean


def test_few_rows_stream_as_far_as_lds_holds_them():
    for T, wide in ((32, 4608), (5, 4608), (4, 19968), (1, 81408)):
        assert experts_plan(T, 2, 8, wide, 2048, True)[0] == 16 and experts_plan(T, 2, 8, wide + 32, 2048, True)[0] == 32


def test_every_tile_that_is_compiled_is_one_that_a_plan_takes():
    """The kernels that the library registers: products of all rows in all four tiles, of experts in those of experts_plan (which
    test_experts_plans_keep_their_bounds holds to them)."""
    with open(ext.LIB_PATH, "rb") as f:
        names = set(re.findall(rb"_ZN3tri17group_tile_kernelINS_9GroupTileILi(\d+)E[^(]*?NS_8GroupMulE(\d)EEELNS_9GroupKindE(\d)E", f.read()))
    got = {tuple(map(int, n)) for n in names}  # (rows of a tile; 16-bit, 4-bit weights, both in 4 bits; rows, parts, gate and up, down)
    want = {(bm, mul, kind) for bm in (32, 64, 128, 256) for mul in (1, 2) for kind in (0, 1)}
    want |= {(bm, 0, kind) for bm in (64, 256) for kind in (2, 3)} | {(bm, 1, kind) for bm in (32, 128, 256) for kind in (2, 3)}
    assert got == want


def test_numbers_beyond_32_bits_are_refused():
    for name in ("top_k", "groups", "top_groups", "group_top"):
        for n in (2 ** 32 + 1, -2 ** 32 + 1, 2 ** 31):
            with pytest.raises(ValueError):
                blocks.Router(**{"top_k": 1, name: n})
    p = ext.route_params(3, sigmoid=True, groups=4, top_groups=2, group_top=2, renormalize=False, scale=0.5)
    assert [getattr(p, f[0]) for f in p._fields_] == [3, 1, 4, 2, 2, 0, 0.5]
