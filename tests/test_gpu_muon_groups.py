"""Orthogonalised momentum over more matrices than one workspace holds, which are done in groups one behind the other in the same memory."""
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from polarai_framework_b200.capi import MuonTensor  # noqa: E402
from test_gpu_muon import check, make, step  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def workspace(d, shapes):
    arr = (MuonTensor * len(shapes))()
    for t, (rows, cols) in zip(arr, shapes):
        t.weights, t.gradient, t.momentum, t.matrices, t.rows, t.cols = 1 << 20, 1 << 21, 1 << 22, 1, rows, cols
    return d.lib.cdll.polar_b200_fmuon_workspace_bytes(arr, len(shapes))


@pytest.mark.parametrize("shapes,looked_at", [
    # the border lies within the matrices of one shape
    ([(4096, 4096)] * 14, (0, 10, 11, 12, 13)),
    # behind the first shape, within the second one's, whose rounds go in pairs; the smaller ones, given first, come last
    ([(300, 200)] * 3 + [(4096, 4096)] * 10 + [(4096, 2048)] * 7 + [(60, 60)] * 2, (0, 2, 3, 12, 13, 16, 17, 18, 19, 20, 21))])
def test_groups(d, shapes, looked_at):
    together, largest = workspace(d, shapes), max(workspace(d, [s]) for s in set(shapes))
    # one group would take all of their memory (the shared parts of it are below 16 KB a matrix)
    assert largest <= together <= 3 << 30 and sum(workspace(d, [s]) - (16 << 10) for s in shapes) > 3 << 30
    ts = [make(s, 90 + i) for i, s in enumerate(shapes)]
    decays, scales = [0.01 * i for i in range(len(ts))], [1 + 0.1 * i for i in range(len(ts))]
    new = step(d, ts, weight_decay=decays, scale=scales)
    for i in looked_at:
        check(*new[i], *ts[i], weight_decay=decays[i], scale=scales[i])
    again = step(d, ts, weight_decay=decays, scale=scales)
    assert all(torch.equal(a, b) for x, y in zip(new, again) for a, b in zip(x, y))
