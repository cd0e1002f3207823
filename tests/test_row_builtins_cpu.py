"""What the builtins on rows and weights refuse, without a GPU: statuses of the C ABI, ValueErrors of DeviceBuiltins before anything is
launched (stand-ins for tensors and library), argument patterns by name."""
import ctypes
import math
import types

import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from polarai_framework_b200 import device_builtins  # noqa: E402
from polarai_framework_b200.capi import AdamwOptions, AdamwTensor, Arg  # noqa: E402

P, NULL = 4096, None                                         # an aligned address that nothing is read from


@pytest.fixture(scope="module")
def c():
    ge.build()
    return ge.load_package().lib().cdll


def test_layer_norm_statuses(c):
    f, b = c.polar_b200_flayernorm, c.polar_b200_flayernorm_grad
    assert f(P, P, P, -1.0, 4, 4, P, P, P, None) == 1 and f(P, P, P, float("nan"), 4, 4, P, P, P, None) == 1
    assert f(NULL, P, P, 1e-5, 4, 4, P, P, P, None) == 1 and f(P, P, P, 1e-5, 4, 4, NULL, P, P, None) == 1
    assert f(P, P, P, 1e-5, 1 << 31, 4, P, P, P, None) == 1 and f(P, P, P, 1e-5, 4, (1 << 31) + 1, P, P, P, None) == 1
    assert f(NULL, P, P, 1e-5, 0, 4, P, P, P, None) == 0 and f(NULL, P, P, 1e-5, 4, 0, P, P, P, None) == 0
    for i in range(4):
        a = [P] * 4
        a[i] = NULL
        assert b(a[0], a[1], P, a[2], a[3], 4, 4, P, P, P, NULL, 0, None) == 1
    assert b(P, P, P, P, P, 4, 4, NULL, P, P, NULL, 0, None) == 1
    assert b(NULL, NULL, P, P, P, 4, 0, NULL, P, P, NULL, 0, None) == 0
    need = c.polar_b200_flayernorm_grad_workspace_bytes(5000, 300)
    assert need > 0 and c.polar_b200_flayernorm_grad_workspace_bytes(0, 300) == 0
    assert c.polar_b200_flayernorm_grad_workspace_bytes(1 << 40, 300) == 0
    assert b(P, P, P, P, P, 5000, 300, P, P, P, P, need - 1, None) == 5 and b(P, P, P, P, P, 5000, 300, P, P, P, P + 4, need, None) == 5


def test_log_probability_statuses(c):
    def f(logits=P, rows=4, classes=10, pitch=10, ids=P, kind=2, lp=P, top=0, top_ids=NULL, top_lp=NULL):
        return c.polar_b200_flogprob(logits, rows, classes, pitch, ids, kind, lp, NULL, NULL, top, top_ids, top_lp, None)

    def b(logits=P, rows=4, classes=10, pitch=10, ids=P, kind=2, lse=P, ent=P, g=P, ge=P, out=P + 8192, dpitch=10):
        return c.polar_b200_flogprob_grad(logits, rows, classes, pitch, ids, kind, lse, ent, g, ge, out, dpitch, None)

    for call in (f, b):
        assert call(kind=3) == 1 and call(kind=-1) == 1 and call(pitch=9) == 1 and call(rows=1 << 31) == 1
        assert call(classes=(1 << 31) + 1, pitch=1 << 33) == 1 and call(logits=NULL) == 1 and call(ids=NULL) == 1
        assert call(kind=0, classes=(1 << 24) + 1, pitch=1 << 25) == 1
        assert call(rows=0) == 0
    assert f(top=33, classes=100, pitch=100, top_ids=P) == 1 and f(top=11, top_ids=P) == 1 and f(classes=0, pitch=0) == 1
    assert f(lp=NULL) == 0                                   # nothing is asked for
    assert b(lse=NULL) == 1 and b(ent=NULL) == 1 and b(g=NULL) == 1 and b(out=NULL) == 1 and b(dpitch=9) == 1
    assert b(out=P, dpitch=11) == 1 and b(classes=0, pitch=0, dpitch=0) == 0


def test_adamw_statuses(c):
    def call(tensors, **o):
        arr = (AdamwTensor * len(tensors))()
        for t, given in zip(arr, tensors):
            t.weights, t.gradient, t.first, t.second, t.count = P, P << 8, P << 9, P << 10, 16
            for k, v in given.items():
                setattr(t, k, v)
        opt = AdamwOptions(1e-3, 0.9, 0.999, 1e-8, 1, None)
        for k, v in o.items():
            setattr(opt, k, v)
        return c.polar_b200_fadamw(arr, len(tensors), ctypes.byref(opt), None)

    for k in ("weights", "gradient", "first", "second"):
        assert call([{k: None}]) == 1
    assert call([{"first_scales": P}]) == 1 and call([{"second_scales": P}]) == 1
    assert call([{"count": 1 << 60}]) == 1
    assert call([{}], beta1=1.0) == 1 and call([{}], beta2=-0.1) == 1 and call([{}], eps=-1.0) == 1 and call([{}], beta1=float("nan")) == 1
    assert call([{}], step=0) == 1
    assert c.polar_b200_fadamw(None, 1, ctypes.byref(AdamwOptions(1e-3, 0.9, 0.999, 1e-8, 1, None)), None) == 1
    assert c.polar_b200_fadamw((AdamwTensor * 1)(), 1, None, None) == 1
    assert call([]) == 0 and call([{"count": 0, "weights": None}]) == 0
    # the same tensor twice, overlapping weights, a moment inside another tensor's weights, both moments one
    far = {"weights": P << 11, "first": P << 12, "second": P << 13}
    assert call([{}, {}]) == 1 and call([{}, {**far, "weights": P + 60}]) == 1 and call([{}, {**far, "first": P}]) == 1
    assert call([{"second": P << 9}]) == 1 and call([{}, {**far, "second": (P << 9) - 4}]) == 1
    assert call([{"weights": P << 9}]) == 1
    # a gradient inside another tensor's weights or its own moments, the schedule inside what is written
    for gradient, more in ((P, far), (P + 63, far), (P - 63, far), ((P << 11) + 60, far), (P << 12, far)):
        assert call([{}, {**more, "gradient": gradient}]) == 1 and b"overlaps" in c.polar_b200_last_error()
    assert call([{"gradient": P << 10}]) == 1 and b"overlaps" in c.polar_b200_last_error()
    for schedule in (P, P + 60, P - 4, (P << 9) + 32):
        assert call([{}], schedule=schedule) == 1 and b"overlaps" in c.polar_b200_last_error()


def test_by_name_patterns(c):
    keep = []

    def args(*given):
        arr = (Arg * len(given))()
        for a, x in zip(arr, given):
            if isinstance(x, tuple):
                shape = (ctypes.c_uint64 * len(x))(*x)
                keep.append(shape)
                a.is_tensor, a.tensor.dims, a.tensor.shape, a.tensor.data = 1, len(x), shape, P
            else:
                a.scalar = x
        return arr

    def call(name, *given):
        return c.polar_b200_launch_by_name(name.encode(), args(*given), len(given), None, 0, None)

    x, v, r, s = (6, 8), (8,), (6,), (6, 3)
    bad = {"flayernorm": [(x, v, v, 1e-5, x, r), (x, r, v, 1e-5, x, r, r), (x, v, v, 1e-5, v, r, r), (x, v, v, 1e-5, x, v, r), (x, v, v, v, x, r, r),
                          ((), v, v, 1e-5, x, r, r)],
           "flayernorm_grad": [(x, x, v, r, r, x, v), (x, x, r, r, r, x, v, v), (x, v, v, r, r, x, v, v), (x, x, v, r, r, x, v, r), (x, x, v, v, r, x, v, v)],
           "flogprob": [(x, r, r, r), (x, v, r, r, r), (v, r, r, r, r), (x, r, r, r, r, s, s)],
           "flogprob_top": [(x, r, r, r, r), (x, r, r, r, r, s, x), (x, r, r, r, r, r, r), (x, r, r, r, r, (6, 9), (6, 9))],
           "flogprob_grad": [(x, r, r, x), (x, r, r, v, x), (x, r, r, r, v), (x, r, r, r, r, x), (x, r, r, v, r, r, x)],
           "fadamw": [(x, (2,), 0.9, 0.9, 1e-8, 0.0, x, x), (x, (1,), 0.9, 0.9, 1e-8, 0.0, x, x, x), (x, (2,), 0.9, 0.9, 1e-8, 0.0, x, x, v),
                      (x, (2,), 0.9, 0.9, 1e-8, x, x, x, x)],
           "fadamw8": [(x, (2,), 0.9, 0.9, 1e-8, 0.0, x, x, x), (x, (2,), 0.9, 0.9, 1e-8, 0.0, x, (11,), (1,), (12,), (1,)),
                       (x, (2,), 0.9, 0.9, 1e-8, 0.0, x, (12,), (2,), (12,), (1,))]}
    for name, calls in bad.items():
        for given in calls:
            assert call(name, *given) in (1, 3), (name, given)
    results = {"flayernorm": 3, "flayernorm_grad": 3, "flogprob": 3, "flogprob_top": 5, "flogprob_grad": 1, "fadamw": 3, "fadamw8": 5}
    for name, n in results.items():
        assert c.polar_b200_result_count(name.encode()) == n
    q = args((30, 20, 300), (30, 20, 300), (300,), (600,), (600,), (30, 20, 300), (300,), (300,))
    assert c.polar_b200_launch_workspace_bytes(b"flayernorm_grad", q, 8) == c.polar_b200_flayernorm_grad_workspace_bytes(600, 300)


class FakeTensor:
    is_cuda = True

    def __init__(self, *shape, dtype=torch.float32, device="cuda:0", strides=None):
        self.shape, self.dtype, self.device, self._strides = shape, dtype, device, strides

    def numel(self):
        return math.prod(self.shape)

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return self._strides[i] if self._strides else math.prod(self.shape[i + 1:])

    def is_contiguous(self):
        return self._strides is None

    def data_ptr(self):
        return P


class Recorder:
    def __init__(self):
        self.calls = []

    def call(self, name, *args):
        self.calls.append(name)


@pytest.fixture
def d(monkeypatch):
    monkeypatch.setattr(device_builtins, "_stream", lambda t: 0)
    b = device_builtins.DeviceBuiltins.__new__(device_builtins.DeviceBuiltins)
    b.lib = Recorder()
    b._native = types.SimpleNamespace(**{n: lambda *a: False for n in ("flayernorm", "flayernorm_grad", "flogprob", "flogprob_grad", "fadamw")})
    return b


T = FakeTensor
I64, I32, F16, U8 = torch.int64, torch.int32, torch.float16, torch.uint8


def norm(x=T(6, 8), gamma=T(8), beta=T(8), out=T(6, 8), mean=T(6), rstd=T(6)):
    return lambda d: d.flayernorm(x, gamma, beta, 1e-5, out, mean, rstd)


def norm_grad(g=T(6, 8), x=T(6, 8), gamma=T(8), mean=T(6), rstd=T(6), dx=T(6, 8), dg=T(8), db=T(8)):
    return lambda d: d.flayernorm_grad(g, x, gamma, mean, rstd, dx, dg, db)


def logprob(x=T(6, 8), ids=T(6, dtype=I64), lp=T(6), ent=T(6), lse=T(6), ti=None, tl=None):
    return lambda d: d.flogprob(x, ids, lp, ent, lse, ti, tl)


def logprob_grad(x=T(6, 8), ids=T(6, dtype=I64), lse=T(6), ent=T(6), g=T(6), ge=T(6), dx=T(6, 8)):
    return lambda d: d.flogprob_grad(x, ids, lse, ent, g, ge, dx)


def adamw(w=(T(300),), g=(T(300),), m=(T(300),), v=(T(300),), ms=None, vs=None, **k):
    return lambda d: d.fadamw(w, g, m, v, ms, vs, **k)


Q = (T(300, dtype=U8),)
GOOD = [norm(), norm(gamma=None, beta=None, mean=None, rstd=None), norm(x=T(2, 3, 8), out=T(2, 3, 8)), norm_grad(), norm_grad(gamma=None, dg=None, db=None),
        logprob(), logprob(ids=None, lp=None), logprob(x=T(6, 8, strides=(11, 1))), logprob(ti=T(6, 3, dtype=I64), tl=T(6, 3)),
        logprob(ids=T(6), ti=T(6, 3)), logprob_grad(), logprob_grad(ent=None, ge=None), logprob_grad(dx=T(6, 8, strides=(9, 1))), adamw(),
        adamw(m=Q, v=Q, ms=(T(3),), vs=(T(3),), weight_decay=[0.0]), adamw(schedule=T(2))]
BAD = [norm(x=T(6, 8, dtype=F16)), norm(gamma=T(7)), norm(beta=T(9)), norm(out=T(6, 7)), norm(mean=T(5)), norm(rstd=T(7)), norm(out=T(6, 8, device="cuda:1")),
       norm_grad(g=T(5, 8)), norm_grad(dx=T(6, 9)), norm_grad(gamma=T(6)), norm_grad(mean=T(8)), norm_grad(dg=T(7)), norm_grad(db=T(9)),
       norm_grad(rstd=T(6, device="cuda:1")),
       logprob(x=T(6, 8, strides=(1, 6))), logprob(x=T(6, 8, strides=(7, 1))), logprob(x=T(48)), logprob(ids=T(6, dtype=F16)), logprob(ids=T(5, dtype=I64)),
       logprob(ids=None), logprob(lp=T(5)), logprob(ent=T(7)), logprob(lse=T(1)), logprob(ti=T(6, 3, dtype=I32)), logprob(ti=T(5, 3, dtype=I64)),
       logprob(ti=T(6, 3, dtype=I64), tl=T(6, 4)), logprob(ti=T(18, dtype=I64)), logprob(ids=T(6, dtype=I64, device="cuda:1")),
       logprob_grad(dx=T(6, 7)), logprob_grad(ids=T(6, dtype=F16)), logprob_grad(lse=T(5)), logprob_grad(g=T(5)), logprob_grad(ge=T(5)), logprob_grad(ent=None),
       logprob_grad(ent=T(1)), logprob_grad(dx=T(6, 8, device="cuda:1")),
       adamw(g=(T(299),)), adamw(m=(T(301),)), adamw(v=(T(1),)), adamw(g=()), adamw(m=Q), adamw(m=Q, v=Q, ms=(T(3),)), adamw(m=Q, v=Q, ms=(T(2),), vs=(T(3),)),
       adamw(ms=(T(3),), vs=(T(3),)), adamw(w=(T(300, dtype=F16),)), adamw(weight_decay=[0.1, 0.2]), adamw(schedule=T(3)), adamw(step=-1),
       adamw(g=(T(300, device="cuda:1"),))]


@pytest.mark.parametrize("i", range(len(GOOD)))
def test_what_fits_is_launched(d, i):
    GOOD[i](d)
    assert len(d.lib.calls) == 1


@pytest.mark.parametrize("i", range(len(BAD)))
def test_what_does_not_fit_is_a_value_error(d, i):
    with pytest.raises(ValueError):
        BAD[i](d)
    assert d.lib.calls == []
