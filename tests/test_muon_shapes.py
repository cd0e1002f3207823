"""Gradients and momenta of fmuon have the shape of their weights: as many elements of another shape are other matrices, which are refused."""
import ctypes
import types

import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from polarai_framework_b200 import device_builtins  # noqa: E402
from polarai_framework_b200.capi import Arg  # noqa: E402
from test_muon_cpu import P, Stand  # noqa: E402

# weights, and what has as many elements
OTHERS = [((20, 30), (30, 20)), ((20, 30), (600,)), ((20, 30), (600, 1)), ((20, 30), (2, 10, 30)), ((3, 20, 30), (3, 30, 20)), ((3, 20, 30), (30, 20, 3)), ((4, 20, 30), (2, 40, 30))]
SAME = [((20, 30), (1, 20, 30)), ((2, 3, 20, 30), (6, 20, 30)), ((6, 20, 30), (2, 3, 20, 30))]


def by_name(c, weights, gradient, momentum):
    given, keep = (gradient, (2,), 0.95, 1.0, 5.0, 0.0, 1.0, weights, momentum), []
    arr = (Arg * len(given))()
    for i, (a, x) in enumerate(zip(arr, given)):
        if isinstance(x, tuple):
            keep.append((ctypes.c_uint64 * len(x))(*x))
            a.is_tensor, a.tensor.dims, a.tensor.shape, a.tensor.data = 1, len(x), keep[-1], (i + 1) << 24   # (addresses that nothing is read from)
        else:
            a.scalar = x
    return c.polar_b200_launch_by_name(b"fmuon", arr, len(given), None, 0, None)


def test_by_name():
    ge.build()
    c = ge.load_package().lib().cdll
    for w, x in OTHERS:
        assert by_name(c, w, x, w) == by_name(c, w, w, x) == 3
    for w, x in SAME:                                        # (what is not refused needs a GPU from there on)
        assert by_name(c, w, x, w) != 3 and by_name(c, w, w, x) != 3


def test_device_builtins_refuse_before_a_launch(monkeypatch):
    d = object.__new__(device_builtins.DeviceBuiltins)
    calls = []
    d._native = types.SimpleNamespace(fmuon=lambda *a: False)
    d.lib = types.SimpleNamespace(call=lambda *a: calls.append(a), cdll=types.SimpleNamespace(polar_b200_fmuon_workspace_bytes=lambda *a: 0))
    monkeypatch.setattr(device_builtins, "_stream", lambda t: None)
    for w, x in OTHERS:
        for g, m in ((x, w), (w, x)):
            with pytest.raises(ValueError):
                d.fmuon([Stand(*w)], [Stand(*g)], [Stand(*m)])
    assert not calls
    for w, x in SAME:
        d.fmuon([Stand(*w)], [Stand(*x)], [Stand(*x)])
    assert len(calls) == len(SAME)


@pytest.mark.gpu
def test_tensors_on_the_gpu():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    from test_gpu_muon import check, make
    d = DeviceBuiltins()
    for w, x in OTHERS:
        a, b = torch.ones(w, device="cuda:0"), torch.ones(x, device="cuda:0")
        for g, m in ((b, a.clone()), (a.clone(), b)):
            kept = m.clone()
            with pytest.raises(ValueError):
                d.fmuon([a], [g], [m], lr=0.5)
            assert (a == 1).all() and torch.equal(m, kept)
    for shape, x in SAME:
        w, g, m = make(shape, 14)
        nw, nm = w.clone(), m.clone()
        d.fmuon([nw], [g.view(x)], [nm.view(x)], lr=0.5)
        check(nw, nm, w, g, m)
