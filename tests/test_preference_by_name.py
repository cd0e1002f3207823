"""The loss of pairs by name and in programs: beside log probabilities of logits on the oracle against differences, on the GPU against the formula in 64 bits."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from oracle import rows_oracle as rows  # noqa: E402
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.program import Program, fuse_program, results_of  # noqa: E402

U = 2.0 ** -24
OPTIONS = (0.5, 0.1, 0.2)                                     # beta, smoothing, margin


def answers_program(tokens, classes, pairs, average, count=0.0):
    """Logits of packed answers, a pair behind another, to the loss and the logits' gradient."""
    p = Program("pairs")
    p.tensor("logits", tokens, classes), p.tensor("dlogits", tokens, classes)
    for t in ("ids", "logp", "entropy", "lse", "ref", "g"):
        p.tensor(t, tokens)
    p.tensor("offsets", 2 * pairs + 1), p.tensor("loss", 3), p.tensor("rewards", 2 * pairs)
    p.inputs, p.outputs = ["logits", "ids", "ref", "offsets"], ["logp", "loss", "rewards", "g", "dlogits"]
    p.constants = {"g": 0.0}
    p.op("flogprob", "logits", "ids", "logp", "entropy", "lse")
    p.op("fpreference_loss", "logp", "ref", "ids", "offsets", *OPTIONS, count, float(average), "loss", "rewards", "g")
    p.op("flogprob_grad", "logits", "ids", "lse", "g", "dlogits")
    return p


def answers(tokens, classes, pairs, seed=0, before=2, behind=3):
    rng = np.random.default_rng(seed)
    f = np.float32
    offsets = np.concatenate([[before], np.sort(rng.integers(before, tokens - behind + 1, 2 * pairs - 1)), [tokens - behind]])
    ids = rng.integers(0, classes, tokens)
    ids[rng.random(tokens) < 0.3] = -1
    logits = rng.standard_normal((tokens, classes)).astype(f)
    return {"logits": logits, "ids": ids.astype(f), "ref": (-np.log(classes) + 0.3 * rng.standard_normal(tokens)).astype(f), "offsets": offsets.astype(f)}


def log_probabilities(d):
    x = d["logits"].astype(np.float64)
    x = x - x.max(1, keepdims=True)
    x = x - np.log(np.exp(x).sum(1, keepdims=True))
    ids = d["ids"].astype(int)
    return np.where(ids >= 0, x[np.arange(len(ids)), np.maximum(ids, 0)], 0.0)


def loss64(d, average, count=0.0):
    return rows.preference_loss64(log_probabilities(d), d["ref"], d["ids"], d["offsets"], *OPTIONS, average, count)


@pytest.mark.parametrize("average", [False, True])
def test_gradient_of_the_logits_against_differences(oracle, average):
    d = answers(25, 5, 3)
    p = answers_program(25, 5, 3, average)
    assert results_of(*p.ops[1]) == ["loss", "rewards", "g"]
    for program in (p, fuse_program(p)):
        ex = OracleExecutor(program, oracle)
        ex.set_inputs(**d)
        ex.run()
        want, rewards, _, _ = loss64(d, average)
        assert np.abs(ex.t["loss"] - want).max() < 1e-6 and np.abs(ex.t["rewards"] - rewards).max() < 1e-5
        for t in range(25):
            for k in range(5):
                shifted = []
                for step in (1e-4, -1e-4):
                    e = {**d, "logits": d["logits"].astype(np.float64)}
                    e["logits"][t, k] += step
                    shifted.append(loss64(e, average)[0][0])
                # differences: third derivatives (below 1) times 2e-9; the gradient: a few roundings of what is below 1
                assert abs((shifted[0] - shifted[1]) / 2e-4 - ex.t["dlogits"][t, k]) < 1e-6


@pytest.mark.gpu
# one CTA, few and many pairs; three kernels, with a warp and with a lane for each sequence
@pytest.mark.parametrize("tokens,pairs", [(30, 2), (1500, 200), (6145, 5), (50000, 300), (30000, 5000)])
@pytest.mark.parametrize("average,count", [(False, 0.0), (True, 0.0), (True, 12345.0)])
def test_on_the_gpu(tokens, pairs, average, count):
    from polarai_framework_b200.program import DeviceExecutor
    d = answers(tokens, 7, pairs, seed=1)
    ex = DeviceExecutor(answers_program(tokens, 7, pairs, average, count))
    ex.set_inputs(**d)
    for _ in range(4):                                       # (from the third run on small programs are graphs)
        ex.run()
        logp = ex.output("logp")
        want, rewards, g, z = rows.preference_loss64(logp, d["ref"], d["ids"], d["offsets"], *OPTIONS, average, count)
        loss, units = ex.output("loss"), count if count > 0 else pairs
        # (as for the direct call: z is rounded once and a pair has some eight operations, the sums some twenty additions; a sigmoid has z's rounding times |z|)
        each = np.maximum(np.logaddexp(0, -z), np.logaddexp(0, z)) + np.abs(z)
        assert abs(loss[0] - want[0]) <= 32 * U * each.sum() / units and abs(loss[1] - want[1]) <= 4 * U
        assert abs(loss[2] - want[2]) <= 32 * U * np.abs(z + OPTIONS[2]).sum() / units
        assert (np.abs(ex.output("rewards") - rewards) <= 2 * U * np.abs(rewards) + 1e-44).all()
        inside = ~np.isnan(g)
        part = np.repeat(np.repeat(np.abs(z), 2), np.diff(d["offsets"]).astype(int))
        whole = np.where(g[inside] != 0, OPTIONS[0] / units, 0.0)
        assert (np.abs(ex.output("g") - g)[inside] <= (16 + part) * U * whole + 1e-44).all() and (ex.output("g")[~inside] == 0).all()
        assert (ex.output("dlogits")[~inside] == 0).all() and np.abs(ex.output("dlogits")).max() > 0
