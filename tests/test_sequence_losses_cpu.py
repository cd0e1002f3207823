"""What the losses over packed sequences refuse, without a GPU, and their oracle against differences and definitions."""
import ctypes
import math
import types

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from oracle import rows_oracle as rows  # noqa: E402
from polarai_framework_b200 import device_builtins  # noqa: E402
from polarai_framework_b200.capi import Arg, PolicyBatch, PolicyOptions, PreferenceOptions  # noqa: E402

P = 1 << 20                                                  # an aligned address that nothing is read from


@pytest.fixture(scope="module")
def c():
    ge.build()
    return ge.load_package().lib().cdll


def at(i):
    return P + (i << 24)


def policy(c, loss=at(9), g=None, ge_=None, batch=True, options=True, ws=None, ws_bytes=0, **k):
    b = PolicyBatch(at(0), at(1), at(2), at(3), at(4), at(5), at(6), 2, 0, 100, 4)
    o = PolicyOptions(0.2, 0.2, 0.1, 0.1, 0.0, 0)
    for name, v in k.items():
        setattr(b if hasattr(b, name) else o, name, v)
    return c.polar_b200_fpolicy_loss(ctypes.byref(b) if batch else None, ctypes.byref(o) if options else None, loss, g, ge_, ws, ws_bytes, None)


def test_policy_statuses(c):
    assert policy(c, batch=False) == 1 and policy(c, options=False) == 1 and policy(c, loss=None) == 1
    for name in ("logprob", "old_logprob", "advantage", "ids", "offsets"):
        assert policy(c, **{name: None}) == 1
    assert policy(c, id_type=3) == 1 and policy(c, id_type=-1) == 1
    assert policy(c, tokens=(1 << 36) + 1) == 1 and policy(c, sequences=1 << 31) == 1
    assert policy(c, id_type=0, tokens=(1 << 24) + 1) == 1 and policy(c, id_type=1, tokens=1 << 31) == 1
    for bad in (-0.1, 1.1, math.nan):
        assert policy(c, clip_low=bad) == 1
    assert policy(c, clip_high=-0.1) == 1 and policy(c, clip_high=math.nan) == 1
    for name in ("kl_weight", "entropy_weight", "count"):
        assert policy(c, **{name: math.nan}) == 1 and policy(c, **{name: math.inf}) == 1
    assert policy(c, count=-1.0) == 1
    assert policy(c, ge_=at(8), entropy=None) == 1
    # what is written overlaps what is read, other than element for element, or itself
    for g in (at(0) + 4, at(4), at(5), at(6), at(6) + 36, at(1) - 4, at(9) + 16):
        assert policy(c, g=g) == 1 and b"overlaps" in c.polar_b200_last_error()
        assert policy(c, ge_=g) == 1
    assert policy(c, g=at(8), ge_=at(8)) == 1 and policy(c, loss=at(3) + 396) == 1 and policy(c, loss=at(6) + 36) == 1
    assert policy(c, g=at(4), advantage_per_token=1, sequences=100) != 0   # (a per-token array: no overlap, but there is no GPU)
    # a workspace that is too small or misplaced
    need = c.polar_b200_fpolicy_loss_workspace_bytes(100000, 4)
    assert need > 100000 // 8 and c.polar_b200_fpolicy_loss_workspace_bytes(4096, 2048) == 0 and c.polar_b200_fpolicy_loss_workspace_bytes(1 << 40, 4) == 0
    assert policy(c, tokens=100000, ws=at(20), ws_bytes=need - 1) == 5 and policy(c, tokens=100000, ws=at(20) + 4, ws_bytes=need) == 5


def preference(c, logprob=at(0), ref=at(1), ids=at(2), offsets=at(3), kind=2, tokens=100, pairs=2, options=True, loss=at(4), rewards=at(5), g=at(6),
               ws=None, ws_bytes=0, **k):
    o = PreferenceOptions(0.1, 0.0, 0.0, 0.0, 0)
    for name, v in k.items():
        setattr(o, name, v)
    return c.polar_b200_fpreference_loss(logprob, ref, ids, offsets, kind, tokens, pairs, ctypes.byref(o) if options else None, loss, rewards, g, ws, ws_bytes,
                                         None)


def test_preference_statuses(c):
    assert preference(c, options=False) == 1 and preference(c, loss=None) == 1
    assert preference(c, logprob=None) == 1 and preference(c, ids=None) == 1 and preference(c, offsets=None) == 1
    assert preference(c, kind=3) == 1 and preference(c, pairs=1 << 30) == 1 and preference(c, tokens=1 << 37) == 1
    assert preference(c, kind=0, tokens=(1 << 24) + 1) == 1 and preference(c, kind=1, tokens=1 << 31) == 1
    for k in ({"beta": math.nan}, {"beta": math.inf}, {"margin": math.nan}, {"smoothing": -0.1}, {"smoothing": 1.5}, {"smoothing": math.nan}, {"count": -1.0}):
        assert preference(c, **k) == 1
    for g in (at(0) + 4, at(1) - 4, at(2), at(3), at(4) + 8, at(5)):
        assert preference(c, g=g) == 1 and b"overlaps" in c.polar_b200_last_error()
    assert preference(c, rewards=at(0)) == 1 and preference(c, rewards=at(3) + 32) == 1 and preference(c, loss=at(5) + 12) == 1
    need = c.polar_b200_fpreference_loss_workspace_bytes(100000, 4)
    assert need > 100000 // 8 and c.polar_b200_fpreference_loss_workspace_bytes(6144, 1024) == 0
    assert preference(c, tokens=100000, ws=at(20), ws_bytes=need - 1) == 5


def test_by_name_patterns(c):
    keep = []

    def call(name, *given):
        arr = (Arg * len(given))()
        for a, x in zip(arr, given):
            if isinstance(x, tuple):
                shape = (ctypes.c_uint64 * len(x))(*x)
                keep.append(shape)
                a.is_tensor, a.tensor.dims, a.tensor.shape, a.tensor.data = 1, len(x), shape, P
            else:
                a.scalar = x
        return c.polar_b200_launch_by_name(name.encode(), arr, len(given), None, 0, None), c.polar_b200_launch_workspace_bytes(name.encode(), arr, len(given))

    t, s, o = (50,), (4,), (5,)
    good = [t, t, t, t, s, t, o, 0.2, 0.2, 0.1, 0.1, 0.0, 0.0, (5,), t, t]
    for i, bad in ((0, s), (3, s), (4, (3,)), (5, (5, 10)), (6, (0,)), (6, (2, 2)), (12, 0.5), (13, s), (14, s), (15, s), (7, t)):
        args = list(good)
        args[i] = bad
        assert call("fpolicy_loss", *args)[0] == 3
    assert call("fpolicy_loss", *good[:-1])[0] == 3
    good = [t, t, t, o, 0.1, 0.0, 0.0, 0.0, 1.0, (3,), s, t]
    for i, bad in ((0, s), (1, s), (3, s), (3, (1, 5)), (8, 2.0), (9, s), (10, o), (11, s), (4, t)):
        args = list(good)
        args[i] = bad
        assert call("fpreference_loss", *args)[0] == 3
    big, offs = (100000,), (5,)
    assert call("fpolicy_loss", big, big, big, big, (9,), big, offs, 0.2, 0.2, 0.1, 0.1, 0.0, 0.0, (5,), big, big)[1] == c.polar_b200_fpolicy_loss_workspace_bytes(100000, 4)
    assert call("fpreference_loss", big, big, big, offs, 0.1, 0.0, 0.0, 0.0, 1.0, (3,), (9,), big)[1] == c.polar_b200_fpreference_loss_workspace_bytes(100000, 2)
    assert c.polar_b200_result_count(b"fpolicy_loss") == 3 and c.polar_b200_result_count(b"fpreference_loss") == 3


class Stand:
    """Stands in for a CUDA tensor."""
    def __init__(self, n, dtype=torch.float32, device="cuda:0", contiguous=True):
        self.n, self.dtype, self.device, self.is_cuda, self.contiguous = n, dtype, device, True, contiguous

    def is_contiguous(self):
        return self.contiguous

    def numel(self):
        return self.n

    def data_ptr(self):
        return P


def stand_in(monkeypatch):
    d = object.__new__(device_builtins.DeviceBuiltins)
    calls = []
    d._native = types.SimpleNamespace(fpolicy_loss=lambda *a: False, fpreference_loss=lambda *a: False)
    d.lib = types.SimpleNamespace(call=lambda *a: calls.append(a))
    monkeypatch.setattr(device_builtins, "_stream", lambda t: None)
    return d, calls


def test_device_builtins_refuse_before_a_launch(monkeypatch):
    d, calls = stand_in(monkeypatch)
    f = lambda n=50, **k: Stand(n, **k)  # noqa: E731
    i = lambda n=50, dtype=torch.int64, **k: Stand(n, dtype, **k)  # noqa: E731

    def policy(lp=f(), old=f(), a=f(4), ids=i(), offsets=i(5), loss=f(5), g=None, h=None, **k):
        return d.fpolicy_loss(lp, old, a, ids, offsets, loss, g, h, **k)
    for bad in ({"lp": f(49)}, {"old": f(51)}, {"a": f(5)}, {"a": f(4), "advantage_per_token": True}, {"ids": i(49)}, {"offsets": i(0)},
                {"offsets": i(5, torch.int32)}, {"ids": i(50, torch.int16), "offsets": i(5, torch.int16)}, {"loss": f(4)}, {"g": f(49)}, {"h": f(49), "entropy": f()},
                {"h": f()}, {"entropy": f(3)}, {"reference": f(3)}, {"lp": f(dtype=torch.float16)}, {"old": f(contiguous=False)}, {"ids": i(contiguous=False)},
                {"g": f(device="cuda:1")}, {"offsets": i(5, device="cuda:1")}):
        with pytest.raises(ValueError):
            policy(**bad)

    def pairs(lp=f(), ids=i(), offsets=i(5), loss=f(3), r=None, g=None, **k):
        return d.fpreference_loss(lp, ids, offsets, loss, r, g, **k)
    for bad in ({"lp": f(49)}, {"ids": i(49)}, {"offsets": i(6)}, {"offsets": i(0)}, {"loss": f(5)}, {"r": f(2)}, {"g": f(4)}, {"reference": f(4)},
                {"offsets": i(5, torch.int32)}, {"g": f(device="cuda:1")}, {"lp": f(dtype=torch.float64)}):
        with pytest.raises(ValueError):
            pairs(**bad)
    assert not calls
    policy(), policy(a=f(50), advantage_per_token=True), pairs(r=f(4), g=f())
    assert [x[0] for x in calls] == ["polar_b200_fpolicy_loss"] * 2 + ["polar_b200_fpreference_loss"]


def small(seed=0, tokens=30, sequences=6):
    rng = np.random.default_rng(seed)
    o = np.concatenate([[2], np.sort(rng.integers(2, tokens - 1, sequences - 1)), [tokens - 2]])
    ids = rng.integers(-1, 3, tokens)
    lp = -np.abs(rng.standard_normal(tokens))
    return lp, lp + 0.05 * rng.standard_normal(tokens), lp + 0.3 * rng.standard_normal(tokens), np.abs(rng.standard_normal(tokens)), rng.standard_normal(tokens), ids, o


@pytest.mark.parametrize("by_sequence", [False, True])
def test_oracle_policy_gradients_are_the_loss_differences(by_sequence):
    lp, old, ref, h, a, ids, o = small()
    run = lambda lp, h: rows.policy_loss64(lp, old, ref, h, a, ids, o, 0.2, 0.3, 0.1, 0.05, by_sequence, True)  # noqa: E731
    _, g, gh, _ = run(lp, h)
    for i in range(2, len(ids) - 2):
        e = np.zeros(len(ids))
        e[i] = 1e-5
        assert abs((run(lp + e, h)[0][0] - run(lp - e, h)[0][0]) / 2e-5 - g[i]) < 1e-8
        assert abs((run(lp, h + e)[0][0] - run(lp, h - e)[0][0]) / 2e-5 - gh[i]) < 1e-8
    assert np.isnan(g[:2]).all() and np.isnan(g[-2:]).all()


@pytest.mark.parametrize("average", [False, True])
def test_oracle_preference_gradient_is_the_loss_difference(average):
    lp, _, ref, _, _, ids, o = small(1)
    run = lambda lp: rows.preference_loss64(lp, ref, ids, o, 0.7, 0.1, 0.2, average)  # noqa: E731
    loss, rewards, g, z = run(lp)
    for i in range(2, len(ids) - 2):
        e = np.zeros(len(ids))
        e[i] = 1e-5
        assert abs((run(lp + e)[0][0] - run(lp - e)[0][0]) / 2e-5 - g[i]) < 1e-8
    # a pair by hand
    s = [sum(lp[t] - ref[t] for t in range(o[k], o[k + 1]) if ids[t] >= 0) / (max(sum(ids[t] >= 0 for t in range(o[k], o[k + 1])), 1) if average else 1)
         for k in range(6)]
    assert np.allclose(rewards, 0.7 * np.array(s), rtol=1e-6)
