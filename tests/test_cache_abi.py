"""Argument checks of the tri_cache_* entry points, on the CPU: nothing is launched."""
import ctypes

import pytest
import torch

from trinity_amd import blocks, ext

NULL, DTYPE, SHAPE, STRIDE, ALIGN, UNSUPPORTED = -1, -2, -3, -4, -5, -6
B, S, Hq, Hkv, D, L = 3, 5, 6, 2, 128, 40


def _h(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def _four(b=B, h=Hkv, rows=L, d=D):
    return _h(b, h, rows, d // 2, dtype=torch.uint8), _h(b, h, rows, d // 32, dtype=torch.uint8)


def _params(**kw):
    p = ext.cache_params(kw.pop("batch", B), kw.pop("n_kv_heads", Hkv), kw.pop("head_dim", D), kw.pop("seq", S),
                         kw.pop("kv_len", L), n_q_heads=kw.pop("n_q_heads", Hq))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _attend(p=None, **kw):
    a = dict(q=_h(B * S, Hq * D), k_cache=_h(B, Hkv, L, D), k_scales=None, v_cache=_h(B, Hkv, L, D), v_scales=None,
             lens=None, scratch=None, lse=None, out=_h(B * S, Hq * D))
    a.update(kw)
    return ext.cache_attention(*a.values(), _params() if p is None else p, validate_only=True)


def _append(p=None, **kw):
    c, x = _four()
    a = dict(k=_h(B * S, Hkv * D), v=_h(B * S, Hkv * D), k_cache=c, k_scales=x, v_cache=c.clone(), v_scales=x.clone(), lens=None)
    a.update(kw)
    return ext.cache_append(*a.values(), _params() if p is None else p, validate_only=True)


def _read(p=None, **kw):
    c, x = _four()
    a = dict(k_cache=c, k_scales=x, v_cache=c.clone(), v_scales=x.clone(), lens=None, k=_h(B, Hkv, S, D), v=_h(B, Hkv, S, D))
    a.update(kw)
    return ext.cache_read(*a.values(), _params() if p is None else p, validate_only=True)


def test_calls_that_are_accepted():
    c, x = _four()
    four = dict(k_cache=c, k_scales=x, v_cache=c, v_scales=x)
    lens = torch.zeros(B, dtype=torch.int32)
    assert _attend() == _attend(**four) == _attend(lens=lens) == _append() == _read() == 0
    assert _attend(lse=torch.zeros(B, Hq, S)) == 0
    assert _attend(scratch=_h(0, dtype=torch.uint8)) == 0
    bf = torch.bfloat16
    assert _attend(q=_h(B * S, Hq * D, dtype=bf), out=_h(B * S, Hq * D, dtype=bf), **four) == 0
    assert _append(k_cache=_h(B, Hkv, L, D), v_cache=_h(B, Hkv, L, D), k_scales=None, v_scales=None, lens=lens) == 0
    blhd = _h(B, L, Hkv, D).transpose(1, 2)  # heads of a position next to one another
    assert _attend(k_cache=blhd, v_cache=blhd) == 0
    assert _append(k_cache=blhd, v_cache=blhd, k_scales=None, v_scales=None) == 0
    qkv = _h(B * S, (Hq + 2 * Hkv) * D)
    assert _attend(q=qkv[:, :Hq * D]) == _append(k=qkv[:, Hq * D:(Hq + Hkv) * D], v=qkv[:, (Hq + Hkv) * D:]) == 0
    shared = _h(1, Hkv, L, D).expand(B, Hkv, L, D)  # one cache read by all sequences
    assert _attend(k_cache=shared, v_cache=shared) == 0
    one = _params(batch=1)
    assert _attend(one, q=_h(S, Hq * D), out=_h(S, Hq * D), k_cache=_h(Hkv, L, D), v_cache=_h(Hkv, L, D)) == 0
    # nothing to do: no tokens, no sequences
    none = _params(seq=0)
    assert _attend(none, q=_h(0, Hq * D), out=_h(0, Hq * D)) == _append(none, k=_h(0, Hkv * D), v=_h(0, Hkv * D)) == 0
    zero = _params(batch=0)
    e, s = _four(b=0)
    assert _attend(zero, q=_h(0, Hq * D), out=_h(0, Hq * D), k_cache=e, k_scales=s, v_cache=e, v_scales=s) == 0
    assert _attend(_params(kv_len=0), k_cache=_h(B, Hkv, 0, D), v_cache=_h(B, Hkv, 0, D)) == 0


def test_parameters():
    assert ext.lib().tri_validate_cache_attention(*[None] * 10) == NULL
    for kw, want in [(dict(head_dim=96), UNSUPPORTED), (dict(n_q_heads=5), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(batch=-1), SHAPE),
                     (dict(seq=-1), SHAPE), (dict(kv_len=-1), SHAPE), (dict(kv_len=L + 1), SHAPE), (dict(scale=0.0), UNSUPPORTED),
                     (dict(scale=float("nan")), UNSUPPORTED), (dict(scale=float("inf")), UNSUPPORTED), (dict(window=-1), SHAPE),
                     (dict(sinks=-1), SHAPE), (dict(window=4, causal=0), UNSUPPORTED), (dict(kv_len=1 << 30), UNSUPPORTED),
                     (dict(seq=1 << 28), UNSUPPORTED)]:
        assert _attend(_params(**kw)) == want, kw
        if ext.lib().tri_cache_scratch_bytes(ctypes.byref(_params(**kw)), 0) >= 0:
            assert kw == dict(kv_len=L + 1)
    assert _attend(_params(window=1 << 30, sinks=(1 << 31) - 1)) == 0
    with pytest.raises(TypeError):
        ext.native().cache_scratch_bytes(ext.attn_params(2, 2, 64, 1), 0)


def test_row_strides_of_2_30():
    p, q = _params(batch=1, n_kv_heads=1, n_q_heads=1, seq=1, kv_len=1), _h(1, D)
    for rows, want in ((1, 0), (2, UNSUPPORTED)):  # one row has none
        near = _h(1, 1, rows, D)
        far = ext.as_tri(near)
        far.stride[2] = 1 << 30
        assert _attend(p, q=q, out=q, k_cache=near, v_cache=near) == 0
        assert _attend(p, q=q, out=q, k_cache=far, v_cache=near) == _attend(p, q=q, out=q, k_cache=near, v_cache=far) == want
        far.stride[2] = (1 << 30) - 8
        assert _attend(p, q=q, out=q, k_cache=far, v_cache=near) == 0


def test_more_heads_than_a_launch_has_workgroups():
    many = _params(batch=1 << 23, n_kv_heads=2, n_q_heads=2, seq=1)
    assert _attend(many) == UNSUPPORTED
    assert ext.lib().tri_cache_scratch_bytes(ctypes.byref(many), 0) == UNSUPPORTED
    assert _attend(_params(batch=(1 << 23) - 1, n_kv_heads=2, n_q_heads=2, seq=1)) == SHAPE


def test_attention_tensors():
    c, x = _four()
    assert _attend(q=None) == _attend(k_cache=None) == _attend(v_cache=None) == _attend(out=None) == NULL
    assert _attend(k_cache=c, k_scales=x, v_cache=_h(B, Hkv, L, D)) == NULL            # one format
    assert _attend(q=_h(B * S, Hq * D).float()) == DTYPE
    assert _attend(out=_h(B * S, Hq * D, dtype=torch.bfloat16)) == DTYPE
    assert _attend(k_cache=_h(B, Hkv, L, D, dtype=torch.bfloat16)) == DTYPE
    assert _attend(k_cache=c, v_cache=c) == DTYPE                                      # codes without their scales
    assert _attend(k_cache=_h(B, Hkv, L, D), k_scales=x, v_cache=c, v_scales=x) == DTYPE
    assert _attend(q=_h(B * S - 1, Hq * D)) == _attend(out=_h(B * S, Hq * D - 8)) == SHAPE
    assert _attend(k_cache=_h(B, Hkv, L - 1, D)) == _attend(v_cache=_h(B - 1, Hkv, L, D)) == SHAPE
    assert _attend(v_cache=_h(B, Hkv, L + 1, D)) == SHAPE                              # caches of one length
    assert _attend(k_cache=_h(Hkv, L, D), v_cache=_h(Hkv, L, D)) == SHAPE
    assert _attend(k_cache=c, k_scales=x[:, :, :, :2], v_cache=c, v_scales=x) == SHAPE
    assert _attend(k_cache=c, k_scales=x[:, :, 1:], v_cache=c, v_scales=x) == SHAPE
    assert _attend(lens=torch.zeros(B, dtype=torch.int64).view(torch.int32)) == SHAPE  # (twice as many)
    assert _attend(lens=torch.zeros(B, dtype=torch.float32)) == DTYPE
    assert _attend(lens=torch.zeros(2 * B, dtype=torch.int32)[::2]) == STRIDE
    assert _attend(k_cache=_h(B, Hkv, L, 2 * D)[..., ::2]) == STRIDE
    assert _attend(k_cache=_h(B, Hkv, L, D + 4)[..., :D]) == STRIDE
    wide = _h(B, Hkv, L, D // 2 + 8, dtype=torch.uint8)[..., :D // 2]
    assert _attend(k_cache=wide, k_scales=x, v_cache=c, v_scales=x) == STRIDE
    odd = _h(B, Hkv, L, 5, dtype=torch.uint8)[..., :4]
    assert _attend(k_cache=c, k_scales=odd, v_cache=c, v_scales=x) == STRIDE
    off = _h(B * S * Hq * D + 8)[4:-4].view(B * S, Hq * D)
    assert _attend(q=off) == _attend(out=off) == ALIGN
    assert _attend(k_cache=c, k_scales=_h(B * Hkv * L * 4 + 4, dtype=torch.uint8)[2:-2].view(B, Hkv, L, 4), v_cache=c, v_scales=x) == ALIGN
    assert _attend(lse=torch.zeros(B, Hq, S + 1)) == _attend(lse=torch.zeros(B * Hq, S)) == SHAPE
    assert _attend(lse=_h(B, Hq, S)) == DTYPE
    assert _attend(lse=torch.zeros(B, S, Hq).transpose(1, 2)) == STRIDE
    raw = _h(1 << 12, dtype=torch.uint8)
    at = (-raw.data_ptr()) % 256
    assert _attend(scratch=raw[at:]) == 0 and _attend(scratch=raw[at + 16:]) == ALIGN
    assert _attend(scratch=_h(1 << 12, dtype=torch.float32)) == _attend(scratch=_h(1 << 12)) == DTYPE


def test_append_tensors():
    c, x = _four()
    assert _append(k=None) == _append(v_cache=None) == _append(v_scales=None) == NULL
    assert _append(k=_h(B * S, Hkv * D + 8)) == SHAPE
    assert _append(v=_h(B * S, Hkv * D, dtype=torch.bfloat16)) == DTYPE
    assert _append(k_cache=c[:1].expand(B, Hkv, L, D // 2)) == STRIDE                  # sequences that share rows
    assert _append(k_scales=x[:, :1].expand(B, Hkv, L, D // 32)) == STRIDE
    assert _append(k_cache=c[:, :, :1].expand(B, Hkv, L, D // 2)) == STRIDE


def test_written_rows_that_share_memory():
    """No two dimensions step over one another's rows, whatever their order."""
    some = _h(2 * B * Hkv * L * D)
    lay = lambda *strides: _append(k_cache=some.as_strided((B, Hkv, L, D), strides + (1,)), v_cache=_h(B, Hkv, L, D), k_scales=None,
                                   v_scales=None)
    assert lay(Hkv * L * D, L * D, D) == lay(D, B * D, B * Hkv * D) == lay(L * Hkv * D, D, Hkv * D) == 0
    assert lay(D, D, D) == lay(Hkv * L * D, (L - 1) * D, D) == lay((Hkv * L - 1) * D, L * D, D) == STRIDE
    assert lay(D, B * D - 8, B * Hkv * D) == lay(L * D, L * D, D) == STRIDE
    both = _h(B, L, Hkv, 2, D)  # k and v side by side
    k, v = (both[:, :, :, i].transpose(1, 2) for i in range(2))
    assert _append(k_cache=k, v_cache=v, k_scales=None, v_scales=None) == 0


def test_read_tensors():
    assert _read(k=None) == _read(v=None) == NULL
    assert _read(k=_h(B, Hkv, S + 1, D)) == _read(v=_h(B, Hkv, L, D)) == SHAPE
    assert _read(v=_h(B, Hkv, S, D, dtype=torch.bfloat16)) == DTYPE
    assert _read(k=_h(1, Hkv, S, D).expand(B, Hkv, S, D)) == STRIDE
    assert _read(k=_h(B, S, Hkv, D).transpose(1, 2)) == 0


def test_scratch_sizes():
    size = lambda four, **kw: ext.cache_scratch_bytes(_params(**kw), four)
    assert size(False, seq=0) == size(True, batch=0) == size(False, kv_len=0) == 0
    assert size(False, batch=1, seq=1, kv_len=32768) > 0 and size(True, batch=1, seq=1, kv_len=32768) > 0
    assert size(True, batch=1, seq=1, kv_len=1 << 29, window=64) <= size(True, batch=1, seq=1, kv_len=1 << 29)


def test_class_refuses():
    op = blocks.CachedAttention(Hq, Hkv, D)
    with pytest.raises(ValueError):
        op.attend(_h(B * S + 1, Hq * D), _h(B, Hkv, L, D), _h(B, Hkv, L, D))
    with pytest.raises(ext.TrinityError):
        blocks.CachedAttention(Hq, Hkv, 96).attend(_h(B * S, Hq * 96), _h(B, Hkv, L, 96), _h(B, Hkv, L, 96))
    with pytest.raises(ext.TrinityError):
        blocks.CachedAttention(Hq, Hkv, D, causal=False, window=8).attend(_h(B * S, Hq * D), _h(B, Hkv, L, D), _h(B, Hkv, L, D))
    for call in (lambda: op.attend(_h(B * S, Hq * D), _h(B, Hkv, L, D), _h(B, Hkv, L, D)),             # host memory
                 lambda: op.append(_h(B * S, Hkv * D), _h(B * S, Hkv * D), _h(B, Hkv, L, D), _h(B, Hkv, L, D)),
                 lambda: op.read(_h(B, Hkv, L, D), _h(B, Hkv, L, D)),
                 lambda: ext.cache_append(_h(B * S, Hkv * D), _h(B * S, Hkv * D), _h(B, Hkv, L, D), None, _h(B, Hkv, L, D), None,
                                          None, _params()),
                 lambda: op.attend(_h(B * S, Hq * D), _h(B, Hkv, L, D), _h(B, Hkv, L, D), kv_len=1 << 40)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        op.attend(None, _h(B, Hkv, L, D), _h(B, Hkv, L, D))
    with pytest.raises(TypeError):
        op.append(_h(B * S, Hkv * D), _h(B * S, Hkv * D), None, None)
    with pytest.raises(ValueError):
        op.read(_h(B, Hkv, L, D), _h(B, Hkv, L, D), dtype=torch.bfloat16)
    c, x = _four()
    with pytest.raises(ValueError):
        op.read(c, c, x, x, dtype=torch.float32)
    codes, scales = op.make_cache(2, Hkv, 7, D, "cpu")
    assert codes.shape == (2, Hkv, 7, 64) and scales.shape == (2, Hkv, 7, 4)
