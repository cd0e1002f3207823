"""What fuse_program has to leave alone: products beside exchanges of their operands or results, results that an update reads in place."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.program import Program, fuse_program  # noqa: E402


def both(oracle, p, inputs):
    """The outputs of the program as it is and fused; an exchange doubles what it is given, as a second rank with the same would."""
    out = []
    for q in (p, fuse_program(p)):
        ex = OracleExecutor(q, oracle, allreduce=lambda t: np.multiply(t, 2, out=t))
        ex.set_inputs(**{k: v.copy() for k, v in inputs.items()})
        ex.run()
        out.append({n: np.array(ex.t[n]) for n in p.outputs})
    return out


def square(name, tensors, inputs, outputs):
    p = Program(name)
    for n in tensors:
        p.tensor(n, 4, 4)
    p.inputs, p.outputs = list(inputs), list(outputs)
    return p


def values(*names):
    rng = np.random.default_rng(len(names))
    return {n: rng.standard_normal((4, 4)).astype(np.float32) for n in names}


@pytest.mark.parametrize("exchanged", ["Z", "X", "W"])
def test_an_exchange_between_a_product_and_its_sigmoid(oracle, exchanged):
    # of the product itself, or of an operand that the product has read before
    p = square("exchange", "XWZH", "XW", "H")
    p.op("fmatmul_f_f", "X", "W", "Z")
    p.op("ALLREDUCE", exchanged)
    p.op("fsigmoid", "Z", "H")
    plain, fused = both(oracle, p, values("X", "W"))
    assert np.array_equal(plain["H"], fused["H"])
    assert [k for k, _ in fuse_program(p).ops] == ["fmatmul_f_f", "ALLREDUCE", "fsigmoid"]


def test_an_exchange_of_something_else_is_no_obstacle(oracle):
    p = square("other", "XWZHG", "XWG", "HG")
    p.op("fmatmul_f_f", "X", "W", "Z")
    p.op("ALLREDUCE", "G")
    p.op("fsigmoid", "Z", "H")
    assert [k for k, _ in fuse_program(p).ops] == ["ALLREDUCE", "fmatmul_f_f_sigmoid"]
    plain, fused = both(oracle, p, values("X", "W", "G"))
    assert all(np.array_equal(plain[n], fused[n]) for n in "HG")


def test_an_update_reads_its_moments_in_place(oracle):
    # the last argument of fadamw is a result that the step reads first: the product that made it stays
    p = square("moments", "XWZHGUm", "XWGUm", "HU")
    p.tensor("schedule", 2)
    p.inputs.append("schedule")
    p.op("fmatmul_f_f", "X", "W", "Z")
    p.op("fsigmoid", "Z", "H")
    p.op("fadamw", "G", "schedule", 0.9, 0.999, 1e-8, 0.0, "U", "m", "Z")
    given = {n: np.abs(v) for n, v in values("X", "W", "G", "U", "m").items()}
    plain, fused = both(oracle, p, {**given, "schedule": np.array([1, 1e-2], np.float32)})
    assert all(np.array_equal(plain[n], fused[n]) for n in "HU")
    assert [k for k, _ in fuse_program(p).ops] == [k for k, _ in p.ops]
