"""A policy step after one whose sequences held more of the rows: what the rows outside the sequences had for a gradient then is no part of this step's."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.program import fuse_program, norm_policy_program  # noqa: E402
from test_norm_policy import OPTIONS, begin, data  # noqa: E402

GRADIENTS = ("dW1", "dW2", "dgamma", "dbeta", "loss")


def batches(batch, sequences, *sizes):
    """Two batches, of which the second has fewer rows in its sequences, with actions in the rows around them."""
    full, short = data(batch, sequences, *sizes, seed=5), data(batch, sequences, *sizes, seed=6)
    full["offsets"] = np.linspace(0, batch, sequences + 1).astype(int).astype(np.float32)
    short["offsets"] = np.linspace(batch // 4, batch // 2, sequences + 1).astype(int).astype(np.float32)
    for d in (full, short):
        d["actions"] = np.abs(d["actions"])
    return full, short


def steps(make, given):
    ex = make()
    for d in given:
        begin(ex, d)                                         # (weights and data: the same each time, but for what the program keeps by itself)
        ex.run()
    return ex


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("by_sequence", [False, True])
def test_on_the_oracle(oracle, by_sequence, fused):
    full, short = batches(24, 3, 5, 6, 4)
    p = norm_policy_program(24, 3, 5, 6, 4, by_sequence=by_sequence, **OPTIONS)
    make = lambda: OracleExecutor(fuse_program(p) if fused else p, oracle)  # noqa: E731
    after, alone = steps(make, (full, short)), steps(make, (short,))
    for n in GRADIENTS:
        assert np.array_equal(after.t[n], alone.t[n]), n
    assert (alone.t["dZ2"][:6] == 0).all() and (alone.t["dZ2"][12:] == 0).all() and (alone.t["dZ2"][6:12] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("shape", [(24, 3, 5, 6, 4), (9001, 300, 31, 200, 300)])
def test_on_the_gpu(shape, fused):
    from polarai_framework_b200.program import DeviceExecutor
    batch, sequences, *sizes = shape
    full, short = batches(batch, sequences, *sizes)
    p = norm_policy_program(batch, sequences, *sizes, by_sequence=True, **OPTIONS)
    make = lambda: DeviceExecutor(fuse_program(p) if fused else p)  # noqa: E731
    after, alone = steps(make, (full, full, full, short)), steps(make, (short,))
    for n in GRADIENTS:
        assert np.array_equal(after.output(n), alone.output(n)), n
