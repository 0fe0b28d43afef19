"""Argument checks of the tri_fp4_*, tri_route and tri_experts_* entry points and of the classes over them, on the CPU: nothing is
launched."""
import copy
import math
import pickle

import pytest
import torch

from trinity_amd import blocks, ext

NULL, DTYPE, SHAPE, STRIDE, ALIGN, UNSUPPORTED = -1, -2, -3, -4, -5, -6
M, K, N = 5, 96, 24
T, E, TOP, W, F = 6, 4, 2, 64, 96
BF = torch.bfloat16


def _h(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def _b(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


def _rows(read=False, **kw):
    a = dict(x=_h(M, K), codes=_b(M, K // 2), scales=_b(M, K // 32))
    a.update(kw)
    if read:
        return ext.fp4_dequantize(a["codes"], a["scales"], a["x"], validate_only=True)
    return ext.fp4_quantize(a["x"], a["codes"], a["scales"], validate_only=True)


def _product(**kw):
    a = dict(x=_h(M, K), x_scales=None, w=_b(N, K // 2), w_scales=_b(N, K // 32), workspace=None, out=_h(M, N))
    a.update(kw)
    return ext.fp4_matmul(*a.values(), validate_only=True)


def _route(logits=None, bias=None, ids=None, weights=None, top_k=TOP, t=T, e=E, **p):
    logits = _h(t, e) if logits is None else logits
    ids = torch.zeros(t, max(top_k, 0), dtype=torch.int32) if ids is None else ids
    weights = torch.zeros(t, max(top_k, 0)) if weights is None else weights
    return ext.route(logits, bias, ids, weights, ext.route_params(top_k, **p), validate_only=True)


def _experts(four=False, **kw):
    w = lambda rows, k: (_b(E, rows, k // 2), _b(E, rows, k // 32)) if four else (_h(E, rows, k), None)
    (g, gs), (u, us), (d, ds) = w(F, W), w(F, W), w(W, F)
    raw = _b(ext.experts_workspace_bytes(T, TOP, E, W, F) + 256)
    a = dict(x=_h(T, W), ids=torch.zeros(T, TOP, dtype=torch.int32), weights=torch.zeros(T, TOP), gate=g, gate_scales=gs, up=u,
             up_scales=us, down=d, down_scales=ds, workspace=raw[(-raw.data_ptr()) % 256:], out=_h(T, W))
    a.update(kw)
    return ext.experts_ffn(*a.values(), validate_only=True)


@pytest.mark.parametrize("read", [False, True])
def test_rows(read):
    assert _rows(read) == _rows(read, x=_h(M, K, dtype=BF)) == 0
    assert _rows(read, x=_h(M, K + 8)[:, :K], codes=_b(M, 64)[:, :48], scales=_b(M * 5 + 1)[1:].view(M, 5)[:, :3]) == 0
    assert _rows(read, x=None) == _rows(read, codes=None) == _rows(read, scales=None) == NULL
    assert _rows(read, x=_h(M, K, dtype=torch.float32)) == _rows(read, codes=_h(M, K // 2)) == DTYPE
    assert _rows(read, codes=_b(M, K // 2 - 16)) == _rows(read, scales=_b(M + 1, K // 32)) == _rows(read, x=_h(M * K)) == SHAPE
    assert _rows(read, codes=_b(M, K // 2 + 8)[:, :K // 2]) == _rows(read, codes=_b(M, K)[:, ::2]) == STRIDE
    assert _rows(read, scales=_b(1, K // 32).expand(M, K // 32)) == STRIDE
    assert _rows(read, codes=_b(M * K // 2 + 16)[8:-8].view(M, K // 2)) == ALIGN
    assert _rows(read, x=_h(M, 48), codes=_b(M, 24), scales=_b(M, 1)) == UNSUPPORTED  # (no whole blocks)
    assert _rows(read, x=_h(M, 0), codes=_b(M, 0), scales=_b(M, 0)) != 0
    assert _rows(read, x=_h(0, K), codes=_b(0, K // 2), scales=_b(0, K // 32)) == 0
    wide = (1 << 22) + 32
    one = lambda k: _rows(read, x=_h(1, k), codes=_b(1, k // 2), scales=_b(1, k // 32))
    assert one(wide) == UNSUPPORTED and one(wide - 32) == 0


def test_product():
    assert _product() == _product(x=_h(M, K, dtype=BF), out=_h(M, N, dtype=BF)) == 0
    four = dict(x=_b(M, K // 2), x_scales=_b(M, K // 32))
    assert _product(**four) == _product(**four, out=_h(M, N, dtype=BF)) == 0
    assert _product(w_scales=_b(N * 7)[1:-3].view(-1)[:N * 6].view(N, 6)[:, :3]) == 0
    for name in ("x", "w", "w_scales", "out"):
        assert _product(**{name: None}) == NULL
    assert _product(x=_h(M, K, dtype=BF)) == _product(out=_h(M, N, dtype=torch.float32)) == _product(w=_h(N, K // 2)) == DTYPE
    assert _product(x=_b(M, K // 2)) == _product(x_scales=_b(M, K // 32)) == DTYPE      # codes without scales, values with
    assert _product(x=_h(M, K + 32)) == _product(out=_h(M, N + 8)) == _product(w_scales=_b(N, K // 32 + 1)) == SHAPE
    assert _product(x=_b(M, K // 2), x_scales=_b(M + 1, K // 32)) == SHAPE
    assert _product(w=_b(N, K)[:, ::2]) == _product(out=_h(M, N + 4)[:, :N]) == STRIDE
    assert _product(w=_b(N * K // 2 + 16)[8:-8].view(N, K // 2)) == ALIGN
    assert _product(x=_h(M, 48), w=_b(N, 24), w_scales=_b(N, 1)) == UNSUPPORTED
    n = _product(w=_b(20, K // 2), w_scales=_b(20, K // 32), out=_h(M, 20))
    assert n != 0                                                                        # columns by eights
    assert _product(workspace=_h(64)) == DTYPE
    assert _product(x=_h(0, K), out=_h(0, N)) == 0
    far = ext.as_tri(_b(N, K // 2))
    far.stride[0] = 1 << 24
    assert _product(w=far) == UNSUPPORTED
    far.stride[0] = (1 << 24) - 16
    assert _product(w=far) == 0
    many = 1 << 9                                                                        # rows that span 4 GB and more
    far = ext.as_tri(_b(many, K // 2))
    far.stride[0] = 1 << 23
    assert _product(w=far, w_scales=_b(many, K // 32), out=_h(M, many)) == UNSUPPORTED
    with pytest.raises(ext.TrinityError):
        ext.fp4_workspace_bytes(4, 48, 8, False)
    with pytest.raises(ext.TrinityError):
        ext.fp4_workspace_bytes(1 << 30, 64, 1 << 20, False)
    assert ext.fp4_workspace_bytes(0, 64, 8, True) == 0


def test_route():
    assert _route() == _route(logits=_h(T, E, dtype=BF)) == _route(logits=torch.zeros(T, E), bias=torch.zeros(E)) == 0
    assert _route(logits=_h(T, E + 3)[:, :E]) == _route(sigmoid=True, groups=2, top_groups=1, group_top=2) == 0
    assert ext.lib().tri_validate_route(*[None] * 5) == NULL
    assert _route(logits=torch.zeros(T, E, dtype=torch.uint8)) == _route(bias=_h(E)) == _route(weights=_h(T, TOP)) == DTYPE
    assert _route(bias=torch.zeros(E + 1)) == _route(weights=torch.zeros(T, TOP + 1)) == SHAPE
    assert _route(ids=torch.zeros(T + 1, TOP, dtype=torch.int32)) == SHAPE
    assert _route(logits=_h(T, 2 * E)[:, ::2]) == _route(weights=torch.zeros(T, 2 * TOP)[:, :TOP]) == STRIDE
    assert _route(bias=torch.zeros(2 * E)[::2]) == STRIDE
    for p, want in [(dict(top_k=0), SHAPE), (dict(top_k=5), SHAPE), (dict(groups=3), SHAPE), (dict(groups=0), SHAPE),
                    (dict(groups=2, top_groups=3), SHAPE), (dict(groups=4, top_groups=1, top_k=2), SHAPE),
                    (dict(groups=4, top_groups=2, group_top=2), SHAPE), (dict(group_top=2), SHAPE),
                    (dict(groups=2, group_top=3), UNSUPPORTED), (dict(scale=math.inf), UNSUPPORTED),
                    (dict(scale=math.nan), UNSUPPORTED), (dict(e=513), UNSUPPORTED), (dict(e=512, top_k=65), UNSUPPORTED),
                    (dict(e=130, groups=65), UNSUPPORTED), (dict(e=512, top_k=64), 0), (dict(e=512, groups=64, top_groups=64), 0)]:
        assert _route(**p) == want, p
    assert _route(t=0) == 0
    with pytest.raises(ValueError):
        blocks.Router(2, scores="tanh")


@pytest.mark.parametrize("four", [False, True])
def test_experts(four):
    assert _experts(four) == _experts(four, out=_h(T, W + 8)[:, :W]) == 0
    for name in ("x", "ids", "weights", "gate", "up", "down", "workspace", "out"):
        assert _experts(four, **{name: None}) == NULL, name
    if four:
        assert _experts(four, up_scales=None) == _experts(four, down_scales=None) == NULL  # one format
        assert _experts(four, gate=_h(E, F, W // 2)) == DTYPE
        assert _experts(four, up=_b(E, F, W)[:, :, ::2]) == STRIDE
        assert _experts(four, down_scales=_b(E, W, F // 32 + 1)) == SHAPE
        assert _experts(four, x=_h(T, W, dtype=BF), out=_h(T, W, dtype=BF)) == 0
    else:
        assert _experts(four, up_scales=_b(E, F, 2)) == NULL
        assert _experts(four, gate=_h(E, F, W, dtype=BF)) == DTYPE
        assert _experts(four, up=_h(E, F, W + 4)[:, :, :W]) == STRIDE
        assert _experts(four, gate=_h(E * F * W + 8)[4:-4].view(E, F, W)) == ALIGN
        assert _experts(four, up=_h(E, W, F).transpose(1, 2)) == STRIDE                     # the other layout
        both = _h(E, 2 * F, W)
        assert _experts(four, gate=both[:, :F], up=both[:, F:]) == 0
        assert _experts(four, gate=_h(1, F, W).expand(E, F, W)) == 0                        # experts may share a matrix
    assert _experts(four, x=_h(T, W, dtype=torch.float32)) == _experts(four, out=_h(T, W, dtype=BF)) == DTYPE
    assert _experts(four, weights=torch.zeros(T, TOP, dtype=torch.float16)) == DTYPE
    assert _experts(four, x=_h(T + 1, W)) == _experts(four, out=_h(T, W + 8)) == _experts(four, weights=torch.zeros(T, 3)) == SHAPE
    assert _experts(four, ids=torch.zeros(TOP, T, dtype=torch.int32).t()) == STRIDE
    small = _b(256 + 256)
    assert _experts(four, workspace=small[(-small.data_ptr()) % 256:][:256]) not in (0, NULL, DTYPE, SHAPE, STRIDE, ALIGN, UNSUPPORTED)
    raw = _b(1 << 20)
    assert _experts(four, workspace=raw[(-raw.data_ptr()) % 256 + 16:]) == ALIGN
    empty = dict(x=_h(0, W), ids=torch.zeros(0, TOP, dtype=torch.int32), weights=torch.zeros(0, TOP), out=_h(0, W), workspace=None)
    assert _experts(four, **empty) == 0


def test_experts_sizes():
    size = ext.experts_workspace_bytes
    assert size(0, 2, 8, 64, 64) == 0 and size(1, 2, 8, 64, 64) > 0
    for bad in [(-1, 2, 8, 64, 64), (1, 0, 8, 64, 64), (1, 2, 0, 64, 64), (1, 2, 8, 0, 64), (1, 2, 8, 48, 64), (1, 2, 8, 64, 40),
                (1, 65, 80, 64, 64), (1, 2, 513, 64, 64), ((1 << 23) + 1, 2, 8, 64, 64), (1, 2, 8, (1 << 22) + 32, 64),
                (1 << 23, 2, 8, 64, 1 << 16)]:
        with pytest.raises(ext.TrinityError):
            size(*bad)


def test_int32_is_for_the_experts_of_tokens_alone():
    i32 = torch.zeros(T, TOP, dtype=torch.int32)
    for call in (lambda: _experts(weights=i32), lambda: _experts(x=i32), lambda: _route(weights=i32), lambda: _route(logits=i32),
                 lambda: _product(x=i32), lambda: _rows(x=i32),
                 lambda: ext.native().experts_ffn(i32, *[None] * 10, 0), lambda: ext.native().route(i32, None, i32, None, ext.route_params(2), 0),
                 lambda: ext.native().fp4_matmul(i32, *[None] * 5, 0)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(TypeError):  # (another call's parameters)
        ext.native().route_new(_h(T, E), None, ext.attn_params(2, 2, 64, 1), 0)


def test_host_memory_is_refused():
    op, x, (w, ws) = blocks.Fp4Matmul(), _h(M, K), (_b(N, K // 2), _b(N, K // 32))
    ids, p = torch.zeros(T, TOP, dtype=torch.int32), torch.zeros(T, TOP)
    g, d = _h(E, F, W), _h(E, W, F)
    for call in (lambda: op.quantize(x), lambda: op.dequantize(w, ws), lambda: op.run(x, w, ws),
                 lambda: blocks.Fp4Matmul(quantize_x=True).run(x, w, ws), lambda: blocks.Router(2).route(_h(T, E)),
                 lambda: blocks.ExpertsFfn().run(_h(T, W), ids, p, g, g, d),
                 lambda: blocks.RoutedFfnPlan(2).run(_h(T, W), _h(W, E), g, g, d),
                 lambda: blocks.RoutedFfnPlan(2).run(_h(T, W), _h(W, E), g, g, d, norm_w=_h(W)),
                 lambda: op.dequantize(w, ws, torch.float32), lambda: op.run(w, w, ws, x_scales=ws, dtype=torch.float32),
                 lambda: ext.fp4_quantize(x, w, ws), lambda: ext.route(_h(T, E), None, ids, p, ext.route_params(2))):
        with pytest.raises(ValueError):
            call()


def test_objects_can_be_copied_and_pickled():
    for op in (blocks.Fp4Matmul(quantize_x=True), blocks.Router(2, scores="sigmoid", scale=2.5), blocks.ExpertsFfn(),
               blocks.RoutedFfnPlan(2, groups=2, top_groups=1, prenorm=True, eps=1e-5)):
        for other in (copy.copy(op), copy.deepcopy(op), pickle.loads(pickle.dumps(op))):
            assert type(other) is type(op) and vars(other).keys() == vars(op).keys()
            if isinstance(op, blocks.Router):
                assert bytes(other._p) == bytes(op._p)
