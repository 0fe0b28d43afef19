"""blocks.CachedAttention on the CPU: what it owns, and what it hands to the compiled binding (a stand-in of it here, as
nothing may be launched)."""
import copy
import contextlib
import ctypes
import pickle
import random
import threading
import types

import pytest
import torch

from trinity_amd import blocks, ext


class _Binding:
    """cache_attend as the binding has it, without the launches; `meet`: calls wait for one another while they hold their scratch."""

    def __init__(self):
        self.meet, self.held = None, []

    def cache_attend(self, q, k_cache, k_scales, v_cache, v_scales, lens, scratch, out, want_lse, kv_len, params, stream):
        if scratch is None or scratch.numel() < 64:
            return 64
        if self.meet is not None:
            self.meet.wait(timeout=30)
            self.held.append(scratch.data_ptr())
            self.meet.wait(timeout=30)
        return q


def test_calls_in_flight_never_hold_one_buffer(monkeypatch):
    """The binding gives up the interpreter lock between the two launches of a call: what the first leaves in its scratch is
    that call's until the second is behind it."""
    binding = _Binding()
    monkeypatch.setattr(ext, "native", lambda: binding)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    op = blocks.CachedAttention(2, 2, 64)
    q, c = torch.zeros(1, 128), torch.zeros(1, 2, 4, 64)
    op.attend(q, c, c)
    assert len(op._scratch) == 1
    binding.meet = threading.Barrier(3)
    failed = []

    def call():
        try:
            op.attend(q, c, c)
        except Exception as e:  # (a broken barrier, for instance)
            failed.append(e)

    threads = [threading.Thread(target=call) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    assert len(set(binding.held)) == 3
    assert len(op._scratch) == 1  # one of them is kept
    binding.meet = None
    kept = next(iter(op._scratch.values()))
    op.attend(q, c, c)
    assert next(iter(op._scratch.values())) is kept


def test_int32_tensors_are_lengths_alone():
    """They came with the lengths of sequences; every other place of every call refuses them as it did before."""
    i32, h = torch.zeros(0, 64, dtype=torch.int32), torch.zeros(0, 64, dtype=torch.float16)
    w = torch.zeros(64, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        ext.as_tri(i32)
    for call in (lambda x: ext.rmsnorm(x, None, h, validate_only=True), lambda x: ext.native().rmsnorm(x, None, h, 1e-5, 0),
                 lambda x: ext.native().matmul(x, w, None, h, None, 0), lambda x: ext.native().gateup_swiglu(h, w, w, x, None, 0)):
        with pytest.raises(TypeError):
            call(i32)
    cache, lens = torch.zeros(1, 1, 4, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    p = ext.cache_params(1, 1, 64, 0, 4)
    args = [h, cache, None, cache, None, lens, None, None, h]
    assert ext.cache_attention(*args, p, validate_only=True) == 0
    for i in (0, 1, 3, 6, 7, 8):
        with pytest.raises(TypeError):
            ext.cache_attention(*args[:i], i32, *args[i + 1:], p, validate_only=True)
        with pytest.raises(TypeError):
            ext.native().cache_attention(*args[:i], i32, *args[i + 1:], p, 0)


@pytest.mark.parametrize("make", [blocks.CachedAttention, blocks.CachedAttentionPlan, lambda *a, **kw: blocks.AttentionPlan(D=64)])
def test_objects_can_be_copied_and_pickled(make):
    """As parts of an nn.Module are (the earlier plans can); a copy has the same parameters and no buffer of the first."""
    op = make(6, 2, 64, window=7, sinks=3)
    own = getattr(op, "attention", op)
    if hasattr(own, "_p"):
        own._scratch[0] = torch.zeros(8)
    for other in (copy.deepcopy(op), copy.copy(op), pickle.loads(pickle.dumps(op))):
        its = getattr(other, "attention", other)
        if hasattr(own, "_p"):
            assert bytes(its._p) == bytes(own._p)
            assert not its._scratch or its is own
            with pytest.raises(ValueError):  # (host memory)
                its.append(torch.zeros(1, 128).half(), torch.zeros(1, 128).half(), *[torch.zeros(1, 2, 4, 64).half()] * 2)
    assert not hasattr(own, "_p") or own._scratch


def test_sizes_beyond_what_a_launch_counts():
    """Products of batch, tokens and heads up to 2^62: refused from the limit on, and sized below it."""
    size = ext.lib().tri_cache_scratch_bytes
    size.restype = ctypes.c_int64
    rng = random.Random(1)
    cases = [(1 << 15, 1 << 15, 1, 1 << 30, 128), (1, 1 << 29, 1, (1 << 31) - 1, 64), ((1 << 23) - 1, 255, 1, 1 << 23, 128),
             (1, (1 << 27) - 257, 1, 1, 128), (1, (1 << 27) - 256, 1, 1, 128), (1, (1 << 28) - 513, 1, 1, 64), (1, (1 << 28) - 512, 1, 1, 64)]
    for _ in range(5000):
        cases.append((int(2 ** rng.uniform(0, 24)), int(2 ** rng.uniform(0, 30)), int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 11)),
                      rng.choice((64, 128))))
    fits = 0
    for B, S, Hkv, group, D in cases:
        p = ext.cache_params(B, Hkv, D, S, 1000, n_q_heads=Hkv * group)
        ok = B * S * Hkv * group * (D // 8) < (1 << 31) - 4096 and B * Hkv < 1 << 24
        assert (size(ctypes.byref(p), 0) >= 0) == ok, (B, S, Hkv, group, D)
        fits += ok
    assert 500 < fits < len(cases) - 500


def _plan_of_records(monkeypatch):
    """A plan whose steps note the current device (`now`) and launch nothing."""
    now, steps = [0], []
    note = lambda *a, **kw: steps.append(now[0])
    for name in ("matmul", "rmsnorm"):
        monkeypatch.setattr(ext, name, note)
    plan = blocks.CachedAttentionPlan(4, 2, 64, prenorm=True, qknorm=True)
    monkeypatch.setattr(plan.attention, "append", note, raising=False)
    monkeypatch.setattr(plan.attention, "attend", note, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], torch.device(d).index
        yield
        now[0] = before

    monkeypatch.setattr(torch.cuda, "device", device)
    return plan, now, steps


def _on(device, *shape):
    """What the plan's own code looks at of a tensor there."""
    t = torch.zeros(*shape, dtype=torch.float16)
    return types.SimpleNamespace(shape=t.shape, device=torch.device(device), is_cuda=device != "cpu", new_empty=t.new_empty)


def test_plan_refuses_tensors_of_other_devices_before_anything_runs(monkeypatch):
    plan, now, steps = _plan_of_records(monkeypatch)
    at = {"X": (8, 128), "WQ": (128, 256), "WK": (128, 128), "WV": (128, 128), "norm_w": (128,)}
    for device in ("cpu", "cuda:1"):
        for name in at:
            t = {k: _on(device if k == name else "cuda:0", *shape) for k, shape in at.items()}
            with pytest.raises(ValueError):
                plan.run(t["X"], t["WQ"], t["WK"], t["WV"], None, None, None, norm_w=t["norm_w"])
    assert not steps


def test_plan_runs_on_its_tensors_gpu(monkeypatch):
    plan, now, steps = _plan_of_records(monkeypatch)
    now[0] = 0
    for index in (0, 1):
        on = lambda *shape: _on("cuda:%d" % index, *shape)
        del steps[:]
        plan.run(on(8, 128), on(128, 256), on(128, 128), on(128, 128), None, None, None, norm_w=on(128))
        assert steps == [index] * 8 and now[0] == 0  # norm, three products, two norms, append, attention


def test_host_memory_is_refused_before_scratch_is_asked_for():
    """A call that cuts its keys into parts, and one that does not, raise the same."""
    op = blocks.CachedAttention(4, 2, 64)
    for rows in (40, 4000):
        q, c = torch.zeros(1, 256).half(), torch.zeros(1, 2, rows, 64).half()
        assert (ext.cache_scratch_bytes(ext.cache_params(1, 2, 64, 1, rows, n_q_heads=4), False) > 0) == (rows == 4000)
        with pytest.raises(ValueError):
            op.attend(q, c, c)
        assert not op._scratch
