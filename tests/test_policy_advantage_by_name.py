"""Whose the advantages are that the policy loss takes by name and in programs, where a batch has as many sequences as tokens: some of those have several
tokens then and others none, and the size of the advantage cannot tell."""
import ctypes

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from oracle import rows_oracle as rows  # noqa: E402
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.capi import Arg  # noqa: E402
from polarai_framework_b200.program import Program, norm_policy_program  # noqa: E402
from test_norm_policy import OPTIONS, begin, data  # noqa: E402


@pytest.fixture(scope="module")
def c():
    ge.build()
    return ge.load_package().lib().cdll


def test_by_name_patterns(c):
    keep = []

    def call(*given):
        arr = (Arg * len(given))()
        for i, (a, x) in enumerate(zip(arr, given)):
            if isinstance(x, tuple):
                shape = (ctypes.c_uint64 * len(x))(*x)
                keep.append(shape)
                a.is_tensor, a.tensor.dims, a.tensor.shape, a.tensor.data = 1, len(x), shape, (i + 1) << 24   # (addresses that nothing is read from)
            else:
                a.scalar = x
        return (c.polar_b200_launch_by_name(b"fpolicy_loss", arr, len(given), None, 0, None),
                c.polar_b200_launch_workspace_bytes(b"fpolicy_loss", arr, len(given)))

    def args(tokens, sequences, advantages, *told):
        t = (tokens,)
        return t, t, t, t, (advantages,), t, (sequences + 1,), 0.2, 0.2, 0.1, 0.1, 0.0, 0.0, *told, (5,), t, t

    refused = 3
    assert call(*args(12, 12, 12))[0] == refused and b"advantage_per_token" in c.polar_b200_last_error()
    for told in (0.0, 1.0):                                  # what is not refused needs a GPU from there on
        assert call(*args(12, 12, 12, told))[0] != refused
    assert call(*args(50, 4, 4))[0] != refused and call(*args(50, 4, 50))[0] != refused and call(*args(1, 1, 1))[0] != refused
    assert call(*args(50, 4, 4, 0.0))[0] != refused and call(*args(50, 4, 50, 1.0))[0] != refused
    for bad in (args(50, 4, 4, 1.0), args(50, 4, 50, 0.0), args(50, 4, 4, 0.5), args(50, 4, 3, 0.0), args(12, 12, 11, 0.0), args(50, 4, 4, (1,)), args(50, 4, 4, 0.0, 0.0)):
        assert call(*bad)[0] == refused
    assert call(*args(100000, 4, 4, 0.0))[1] == call(*args(100000, 4, 4))[1] == c.polar_b200_fpolicy_loss_workspace_bytes(100000, 4) > 0


def uneven(batch, seed):
    """A batch of as many sequences as rows, some of several rows and some of none."""
    d = data(batch, batch, 5, 6, 4, seed)
    assert len(d["offsets"]) == batch + 1 and 0 in np.diff(d["offsets"]) and np.diff(d["offsets"]).max() > 1
    return d


def want(d, t, by_sequence, per_token=False):
    return rows.policy_loss64(t["logp"], d["old_logp"], d["ref_logp"], t["entropy"], d["advantage"], d["actions"], d["offsets"], *OPTIONS.values(), by_sequence, per_token)


@pytest.mark.parametrize("by_sequence", [False, True])
def test_program_of_as_many_sequences_as_rows(oracle, by_sequence):
    d = uneven(12, 3)
    ex = begin(OracleExecutor(norm_policy_program(12, 12, 5, 6, 4, by_sequence=by_sequence, **OPTIONS), oracle), d)
    ex.run()
    loss, *_ = want(d, ex.t, by_sequence)
    assert np.abs(ex.t["loss"] - loss).max() < 2e-7
    assert abs(loss[0] - want(d, ex.t, by_sequence, True)[0][0]) > 1e-3   # (read one to a row they would be another loss)


def loss_program(tokens, sequences, *told):
    p = Program("loss")
    for n in ("lp", "old", "ref", "entropy", "ids", "g", "ge"):
        p.tensor(n, tokens)
    p.tensor("advantage", tokens if told and told[0] else sequences), p.tensor("offsets", sequences + 1), p.tensor("loss", 5)
    p.inputs, p.outputs = ["lp", "old", "ref", "entropy", "ids", "advantage", "offsets", "g", "ge"], ["loss", "g", "ge"]
    p.op("fpolicy_loss", "lp", "old", "ref", "entropy", "advantage", "ids", "offsets", 0.2, 0.25, 0.1, 0.01, 0.0, 1.0, *told, "loss", "g", "ge")
    return p


def test_oracle_refuses_what_the_size_cannot_tell(oracle):
    ex = OracleExecutor(loss_program(7, 7), oracle)
    ex.set_inputs(**{n: np.zeros(s, np.float32) for n, s in ex.program.tensors.items() if n != "loss"})
    with pytest.raises(ValueError):
        ex.run()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [12, 900, 7001])
@pytest.mark.parametrize("told", [0.0, 1.0])
def test_by_name_on_the_gpu(tokens, told):
    from polarai_framework_b200.program import DeviceExecutor
    from test_gpu_sequence_losses import batch, check
    b = batch(70, tokens, tokens)
    ex = DeviceExecutor(loss_program(tokens, tokens, told))
    advantage = b["token_advantage"] if told else b["advantage"]
    seven = np.full(tokens, 7, np.float32)
    f = lambda v: np.asarray(v, np.float32)  # noqa: E731
    ex.set_inputs(lp=b["logprob"], old=b["old"], ref=b["reference"], entropy=b["entropy"], ids=f(b["ids"]), advantage=f(advantage), offsets=f(b["offsets"]), g=seven, ge=seven)
    ex.run()
    reference = rows.policy_loss64(b["logprob"], b["old"], b["reference"], b["entropy"], advantage, b["ids"], b["offsets"], 0.2, 0.25, 0.1, 0.01, True, bool(told))
    check((ex.output("loss"), ex.output("g"), ex.output("ge"), reference))


@pytest.mark.gpu
@pytest.mark.parametrize("by_sequence", [False, True])
def test_program_on_the_gpu(by_sequence):
    from polarai_framework_b200.program import DeviceExecutor
    d = uneven(40, 4)
    ex = begin(DeviceExecutor(norm_policy_program(40, 40, 5, 6, 4, by_sequence=by_sequence, **OPTIONS)), d)
    ex.run()
    loss, _, _, (size, _) = want(d, {n: ex.output(n) for n in ("logp", "entropy")}, by_sequence)
    assert (np.abs(ex.output("loss") - loss) <= 32 * 2.0 ** -24 * size + 1e-44).all()
