"""fmuon builtins in a row in a program share their launches: as many as one of them takes, where the matrices are of one shape."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from polarai_framework_b200.program import Program  # noqa: E402
from test_gpu_muon import check  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def launches(d, shape, ops, between=False):
    """Runs a program of fmuon builtins, each (weights, momentum factor, nesterov, steps, decay, scale), once: how many launches, and the executor with its data."""
    from polarai_framework_b200.program import DeviceExecutor
    p = Program("updates")
    names = sorted({o[0] for o in ops})
    for n in names:
        for k in ("", "d", "m"):
            p.tensor(k + n, *shape)
    p.tensor("schedule", 2), p.tensor("other", 2)
    p.inputs, p.outputs = [k + n for n in names for k in ("", "d", "m")] + ["schedule"], names
    for i, (n, momentum, nesterov, steps, decay, scale) in enumerate(ops):
        if between and i:
            p.op("fmul", "schedule", "schedule", "other")
        p.op("fmuon", "d" + n, "schedule", momentum, nesterov, steps, decay, scale, n, "m" + n)
    ex = DeviceExecutor(p)
    rng = np.random.default_rng(sum(shape))
    data = {k + n: rng.standard_normal(shape).astype(np.float32) for n in names for k in ("", "d", "m")}
    ex.set_inputs(**data, schedule=np.array([1, 0.5], np.float32))
    before = d.lib.launch_count()
    ex.run()
    count = d.lib.launch_count() - before
    torch.cuda.synchronize()
    assert d.device_status() == 0
    return count, ex, data


# one CTA's matrices; products of clusters; narrow matrices; rounds in pairs
@pytest.mark.parametrize("shape", [(64, 100), (90, 200), (300, 200), (1000, 90), (600, 260)])
def test_in_a_row(d, shape):
    kind = (0.9, 1.0, 5.0)
    one, *_ = launches(d, shape, [("A", *kind, 0.01, 0.7)])
    assert one >= 1 and (one == 1) == (shape in ((64, 100), (90, 200)))
    three, ex, data = launches(d, shape, [("A", *kind, 0.01, 0.7), ("B", *kind, 0.02, 0.8), ("C", *kind, 0.0, 1.0)])
    assert three == one
    for n, decay, scale in (("A", 0.01, 0.7), ("B", 0.02, 0.8), ("C", 0.0, 1.0)):
        w, g, m = (torch.from_numpy(data[k + n]).cuda() for k in ("", "d", "m"))
        check(ex.t[n], ex.t["m" + n], w, g, m, lr=0.5, momentum=0.9, weight_decay=decay, scale=scale)


@pytest.mark.parametrize("shape", [(64, 100), (300, 200)])
def test_what_does_not_share(d, shape):
    kind, rest = (0.9, 1.0, 5.0), (0.01, 0.7)
    one, *_ = launches(d, shape, [("A", *kind, *rest)])
    # another momentum, with and without nesterov, the same matrix once more, something else between them
    for other in ((0.8, 1.0, 5.0), (0.9, 0.0, 5.0)):
        count, ex, data = launches(d, shape, [("A", *kind, *rest), ("B", *other, *rest)])
        assert count == 2 * one
        for n, (momentum, nesterov, _) in (("A", kind), ("B", other)):
            w, g, m = (torch.from_numpy(data[k + n]).cuda() for k in ("", "d", "m"))
            check(ex.t[n], ex.t["m" + n], w, g, m, lr=0.5, momentum=momentum, nesterov=bool(nesterov), weight_decay=rest[0], scale=rest[1])
    assert launches(d, shape, [("A", *kind, *rest), ("A", *kind, *rest)])[0] == 2 * one
    assert launches(d, shape, [("A", *kind, *rest), ("B", *kind, *rest)], between=True)[0] == 2 * one + 1
    # another number of rounds
    few, *_ = launches(d, shape, [("A", 0.9, 1.0, 3.0, *rest)])
    assert launches(d, shape, [("A", *kind, *rest), ("B", 0.9, 1.0, 3.0, *rest)])[0] == one + few
