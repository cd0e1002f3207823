"""What fmuon refuses, without a GPU, and its oracle against the singular value decomposition."""
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
from polarai_framework_b200.capi import Arg, MuonOptions, MuonTensor  # noqa: E402

P = 1 << 22


@pytest.fixture(scope="module")
def c():
    ge.build()
    return ge.load_package().lib().cdll


def tensors(*given):
    arr = (MuonTensor * max(len(given), 1))()
    for t, k in zip(arr, given):
        t.weights, t.gradient, t.momentum, t.matrices, t.rows, t.cols, t.scale = P, P << 1, P << 2, 1, 20, 30, 1.0
        for name, v in k.items():
            setattr(t, name, v)
    return arr


def call(lib, *given, workspace=None, workspace_bytes=0, **o):
    opt = MuonOptions(0.02, 0.95, 1, 5, 3.4445, -4.7750, 2.0315, None)
    for k, v in o.items():
        setattr(opt, k, v)
    return lib.polar_b200_fmuon(tensors(*given), len(given), ctypes.byref(opt), workspace, workspace_bytes, None)


def test_statuses(c):
    assert c.polar_b200_fmuon(tensors({}), 1, None, None, 0, None) == 1
    assert c.polar_b200_fmuon(None, 1, ctypes.byref(MuonOptions(0.02, 0.95, 1, 5, 3.4445, -4.7750, 2.0315, None)), None, 0, None) == 1
    for k in ("weights", "gradient", "momentum"):
        assert call(c, {k: None}) == 1
    for mu in (-0.1, 1.0, math.nan):
        assert call(c, {}, momentum=mu) == 1
    assert call(c, {}, steps=0) == 1 and call(c, {}, steps=33) == 1
    # polynomials under which a singular value passes what the products hold
    for a, b, cc in ((3.4445, 0.0, 0.0), (4.1, -4.775, 2.0), (math.nan, 0.0, 0.0), (1.0, 1.0, 1.0), (3.4445, -4.775, 4.0), (math.inf, 0.0, 0.0)):
        assert call(c, {}, a=a, b=b, c=cc) == 1 and b"1.4" in c.polar_b200_last_error()
    assert call(c, {"rows": (1 << 20) + 1}) == 1 and call(c, {"rows": 32769, "cols": 32769}) == 1 and call(c, {"matrices": 1 << 21}) == 1
    assert call(c) == 0 and call(c, {"rows": 0, "weights": None}) == 0 and call(c, {"matrices": 0}) == 0
    # the same tensor twice, weights that overlap, a momentum or a gradient inside what another writes, the schedule
    far = {"weights": P << 3, "momentum": P << 4}
    assert call(c, {}, {}) == 1 and call(c, {}, {**far, "weights": P + 2396}) == 1 and call(c, {}, {**far, "momentum": P - 4}) == 1
    assert call(c, {"gradient": P}) == 1 and call(c, {"momentum": P << 1}) == 1 and call(c, {}, {**far, "gradient": (P << 2) + 8}) == 1
    assert call(c, {"matrices": 3}, {**far, "weights": P + 7196}) == 1
    for schedule in (P, P - 4, (P << 2) + 2392):
        assert call(c, {}, schedule=schedule) == 1 and b"overlaps" in c.polar_b200_last_error()


def test_workspace(c):
    need = lambda *t: c.polar_b200_fmuon_workspace_bytes(tensors(*t), len(t))  # noqa: E731
    assert need() == 0 and c.polar_b200_fmuon_workspace_bytes(None, 3) == 0
    assert need({"rows": 1 << 21}) == 0                      # refused
    big = {"rows": 1024, "cols": 1024}
    assert 16 * 1024 * 1024 <= need(big) <= 48 * 1024 * 1024
    assert need(*[{**big, "weights": P << (3 + i)} for i in range(3)]) >= 2 * need(big)
    huge = {"rows": 8192, "cols": 8192, "matrices": 50}
    assert need(huge) <= 3 << 30                              # in groups
    one = {"rows": 16384, "cols": 32768}
    assert need(one) > 3 << 30 and need({**one, "matrices": 4}) == need(one)
    n = need(big)
    assert call(c, big, workspace=P << 8, workspace_bytes=n - 1) == 5 and call(c, big, workspace=(P << 8) + 16, workspace_bytes=n) == 5


def test_workspace_of_steps_in_a_row(c):
    """Steps in a row share a workspace: what all of them take together, but no more than a group of them."""
    native = ge.load_package().capi.binding()
    keep = []

    def op(rows, cols):
        given = [(rows, cols), (2,), 0.95, 1.0, 5.0, 0.0, 1.0, (rows, cols), (rows, cols)]
        arr = (Arg * len(given))()
        for a, x in zip(arr, given):
            if isinstance(x, tuple):
                shape = (ctypes.c_uint64 * len(x))(*x)
                keep.append(shape)
                a.is_tensor, a.tensor.dims, a.tensor.shape, a.tensor.data = 1, len(x), shape, P
            else:
                a.scalar = x
        keep.append(arr)
        return b"fmuon", ctypes.addressof(arr), len(given)

    need = lambda *t: c.polar_b200_fmuon_workspace_bytes(tensors(*t), len(t))  # noqa: E731
    for count, rows, cols in ((1, 300, 200), (3, 300, 200), (2, 1024, 4096), (40, 4096, 16384), (40, 8192, 8192), (3, 16384, 32768), (500, 129, 257)):
        got = native.workspace_bytes([op(rows, cols) for _ in range(count)])
        together = need(*[{"rows": rows, "cols": cols}] * count)
        assert together <= got <= max(3 << 30, need({"rows": rows, "cols": cols}))
    # what stands between them has a workspace of its own
    fill = (Arg * 2)()
    shape = (ctypes.c_uint64 * 1)(4)
    fill[0].scalar, fill[1].is_tensor, fill[1].tensor.dims, fill[1].tensor.shape, fill[1].tensor.data = 1.0, 1, 1, shape, P
    apart = native.workspace_bytes([op(300, 200), (b"ffill", ctypes.addressof(fill), 2), op(300, 200)])
    assert apart == need({"rows": 300, "cols": 200})


def test_by_name_patterns(c):
    keep = []

    def by_name(*given):
        arr = (Arg * len(given))()
        for a, x in zip(arr, given):
            if isinstance(x, tuple):
                shape = (ctypes.c_uint64 * len(x))(*x)
                keep.append(shape)
                a.is_tensor, a.tensor.dims, a.tensor.shape, a.tensor.data = 1, len(x), shape, P
            else:
                a.scalar = x
        return c.polar_b200_launch_by_name(b"fmuon", arr, len(given), None, 0, None), c.polar_b200_launch_workspace_bytes(b"fmuon", arr, len(given))

    good = [(20, 30), (2,), 0.95, 1.0, 5.0, 0.0, 1.0, (20, 30), (20, 30)]
    big = [(200, 300), (2,), 0.95, 1.0, 5.0, 0.0, 1.0, (200, 300), (200, 300)]
    assert by_name(*big)[1] == c.polar_b200_fmuon_workspace_bytes(tensors({"rows": 200, "cols": 300}), 1) > 0
    assert by_name(*good)[1] == 0                            # (one CTA's shared memory holds it)
    for i, bad in ((0, (20, 29)), (0, 1.0), (1, (3,)), (3, 0.5), (4, 0.0), (4, 2.5), (4, 33.0), (4, math.nan), (7, (600,)), (8, (20, 31)), (2, (20, 30))):
        args = list(good)
        args[i] = bad
        if i == 7:
            args[0] = args[8] = bad
        assert by_name(*args) == (3, 0)
    assert by_name(*good[:-1]) == (3, 0) and c.polar_b200_result_count(b"fmuon") == 2


class Stand:
    """Stands in for a CUDA tensor."""
    def __init__(self, *shape, dtype=torch.float32, device="cuda:0", contiguous=True):
        self.shape, self.dtype, self.device, self.is_cuda, self.contiguous = shape, dtype, device, True, contiguous

    def is_contiguous(self):
        return self.contiguous

    def numel(self):
        return math.prod(self.shape)

    def data_ptr(self):
        return P


def test_device_builtins_refuse_before_a_launch(monkeypatch):
    d = object.__new__(device_builtins.DeviceBuiltins)
    calls = []
    d._native = types.SimpleNamespace(fmuon=lambda *a: False)
    d.lib = types.SimpleNamespace(call=lambda *a: calls.append(a), cdll=types.SimpleNamespace(polar_b200_fmuon_workspace_bytes=lambda *a: 0))
    monkeypatch.setattr(device_builtins, "_stream", lambda t: None)
    x = Stand(4, 6)
    for w, g, m, k in (([x], [x, x], [x], {}), ([x], [x], [], {}), ([x], [Stand(4, 5)], [x], {}), ([Stand(24)], [Stand(24)], [Stand(24)], {}),
                       ([x], [x], [Stand(4, 6, dtype=torch.bfloat16)], {}), ([x], [Stand(4, 6, contiguous=False)], [x], {}), ([x], [x], [x], {"weight_decay": [0.1, 0.2]}),
                       ([x], [x], [x], {"scale": []}), ([x], [Stand(4, 6, device="cuda:1")], [x], {}), ([x], [x], [x], {"schedule": Stand(3)}),
                       ([x], [x], [x], {"schedule": Stand(2, device="cuda:1")})):
        with pytest.raises(ValueError):
            d.fmuon(w, g, m, **k)
    assert not calls
    d.fmuon([], [], [])
    assert not calls
    d.fmuon([x, Stand(2, 3, 5)], [x, Stand(2, 3, 5)], [x, Stand(2, 3, 5)])
    (name, arr, n, *_), = calls
    assert name == "polar_b200_fmuon" and n == 2 and (arr[1].matrices, arr[1].rows, arr[1].cols) == (2, 3, 5)
    assert arr[0].scale == 1.0
    d.fmuon([Stand(18, 2)], [Stand(18, 2)], [Stand(18, 2)])
    assert calls[-1][1][0].scale == 3.0


@pytest.mark.parametrize("shape", [(5, 9), (9, 5), (6, 6)])
def test_oracle_is_the_polynomial_of_the_singular_values(shape):
    rng = np.random.default_rng(sum(shape))
    w, g, m = (rng.standard_normal(shape) for _ in range(3))
    nw, nm, x = rows.muon64(w, g, m, 0.1, 0.9, True, 5, 0.01, 0.5)
    u = g + float(np.float32(0.9)) * nm
    left, s, right = np.linalg.svd(u, full_matrices=False)
    s = s / np.sqrt((s * s).sum())
    a, b, c = (float(np.float32(v)) for v in (3.4445, -4.7750, 2.0315))
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert np.abs(x - (left * s) @ right).max() < 1e-10
    assert np.allclose(nw, w * (1 - 0.1 * 0.01) - 0.05 * x, atol=1e-7)
    assert np.allclose(nm, 0.9 * m + g, atol=1e-6)
