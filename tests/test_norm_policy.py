"""A policy gradient step made of the builtins - matmul, layer norm, sigmoid, matmul, log probability, policy loss, their gradients,
orthogonalised momentum for the matrices, AdamW for the vectors - as one program: on the oracle against differences, on the GPU against the oracle."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from oracle import rows_oracle as rows  # noqa: E402
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.program import fuse_program, norm_policy_program, results_of  # noqa: E402

OPTIONS = dict(clip_low=0.2, clip_high=0.3, kl_weight=0.1, entropy_weight=0.02)


def data(batch, sequences, n_in, n_hidden, actions, seed=0):
    rng = np.random.default_rng(seed)
    f = np.float32
    picked = rng.integers(0, actions, batch).astype(f)
    picked[::5] = -1
    offsets = np.concatenate([[1], np.sort(rng.integers(1, batch - 1, sequences - 1)), [batch - 1]]).astype(f)
    logp = (-np.log(actions) + 0.2 * rng.standard_normal(batch)).astype(f)
    return {"X": rng.standard_normal((batch, n_in)).astype(f), "actions": picked, "offsets": offsets, "old_logp": logp,
            "ref_logp": (logp + 0.1 * rng.standard_normal(batch)).astype(f), "advantage": rng.standard_normal(sequences).astype(f),
            "W1": (rng.standard_normal((n_in, n_hidden)) / np.sqrt(n_in)).astype(f), "W2": (rng.standard_normal((n_hidden, actions)) / np.sqrt(n_hidden)).astype(f),
            "gamma": (1 + 0.1 * rng.standard_normal(n_hidden)).astype(f), "beta": (0.1 * rng.standard_normal(n_hidden)).astype(f)}


def begin(ex, inputs, lr=1e-2):
    ex.set_inputs(**inputs, schedule=np.array([0, lr], np.float32), tick=np.array([1, 0], np.float32))
    zeros = [n for n in ex.program.inputs if n not in inputs and n not in ("schedule", "tick")]
    if hasattr(ex, "set_zeros"):
        ex.set_zeros(*zeros)
    return ex


def loss64(d, by_sequence):
    e = {k: v.astype(np.float64) for k, v in d.items()}
    z = e["X"] @ e["W1"]
    dev = z - z.mean(1, keepdims=True)
    n = dev / np.sqrt((dev ** 2).mean(1, keepdims=True) + np.float64(np.float32(1e-5))) * e["gamma"] + e["beta"]
    l = 1 / (1 + np.exp(-n)) @ e["W2"]
    l = l - np.log(np.exp(l).sum(1, keepdims=True))
    ids = d["actions"].astype(int)
    logp = np.where(ids >= 0, l[np.arange(len(ids)), np.maximum(ids, 0)], 0.0)
    entropy = -(np.exp(l) * l).sum(1)
    return rows.policy_loss64(logp, d["old_logp"], d["ref_logp"], entropy, d["advantage"], d["actions"], d["offsets"], *OPTIONS.values(), by_sequence)[0]


@pytest.mark.parametrize("by_sequence", [False, True])
def test_gradients_of_the_step_against_differences(oracle, by_sequence):
    d = data(17, 4, 5, 6, 4)
    ex = begin(OracleExecutor(norm_policy_program(17, 4, 5, 6, 4, by_sequence=by_sequence, **OPTIONS), oracle), d)
    ex.run()
    assert np.abs(ex.t["loss"] - loss64(d, by_sequence)).max() < 2e-6
    rng = np.random.default_rng(1)
    for name in ("W1", "W2", "gamma", "beta"):
        grad = ex.t["d" + name]
        for _ in range(8):
            at = tuple(rng.integers(0, s) for s in grad.shape)
            shifted = []
            for step in (1e-3, -1e-3):
                e = {k: v.astype(np.float64) for k, v in d.items()}
                e[name][at] += step
                shifted.append(loss64(e, by_sequence)[0])
            # differences: third derivatives (below 10) times 1.7e-7; the gradient: fp32 sums of a few terms below 1
            assert abs((shifted[0] - shifted[1]) / 2e-3 - grad[at]) < 5e-6


def test_the_fused_form_is_the_same_program(oracle):
    d = data(30, 3, 8, 12, 5)
    plain = norm_policy_program(30, 3, 8, 12, 5, **OPTIONS)
    fused = fuse_program(plain)
    assert "fdense_grad" in [k for k, _ in fused.ops] and results_of(*plain.ops[-3]) == ["W2", "M_W2"]
    a, b = (begin(OracleExecutor(p, oracle), d) for p in (plain, fused))
    for _ in range(3):
        a.run(), b.run()
    assert all(np.array_equal(a.t[n], b.t[n]) for n in plain.outputs)


def test_two_ranks_share_a_batch(oracle):
    # the gradients of two halves with the whole batch's count add up to its own
    d = data(20, 4, 6, 8, 4)
    d["offsets"] = np.array([0, 4, 10, 13, 20], np.float32)
    whole = begin(OracleExecutor(norm_policy_program(20, 4, 6, 8, 4, **OPTIONS), oracle), d)
    whole.run()
    count = float((d["actions"] >= 0).sum())
    halves = []
    for i in range(2):
        rows_of = {k: d[k][10 * i:10 * i + 10] for k in ("X", "actions", "old_logp", "ref_logp")}
        part = {**d, **rows_of, "offsets": d["offsets"][2 * i:2 * i + 3] - 10 * i, "advantage": d["advantage"][2 * i:2 * i + 2]}
        halves.append(begin(OracleExecutor(norm_policy_program(10, 2, 6, 8, 4, count=count, **OPTIONS), oracle), part))
        halves[-1].run()
    for name in ("W1", "W2", "gamma", "beta"):
        assert np.abs(halves[0].t["d" + name] + halves[1].t["d" + name] - whole.t["d" + name]).max() < 16 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("shape", [(33, 5, 20, 36, 7), (257, 20, 784, 512, 10), (9001, 300, 31, 200, 300)])
def test_the_step_on_the_gpu_against_the_oracle(oracle, shape, fused):
    from polarai_framework_b200.program import DeviceExecutor
    batch, sequences, *sizes = shape
    d = data(batch, sequences, *sizes)
    program = norm_policy_program(batch, sequences, *sizes, by_sequence=True, **OPTIONS)
    want, got = begin(OracleExecutor(program, oracle), d), begin(DeviceExecutor(fuse_program(program) if fused else program), d)
    want.run(), got.run()
    for n in ("loss", "logp", "entropy", "dW1", "dW2", "dgamma", "dbeta"):
        a, b = got.output(n).astype(np.float64), want.t[n]
        # gradients: products whose sums agree to 5e-6 of their terms (the matmuls' tolerance), some of which cancel
        assert np.linalg.norm(a - b) <= 1e-4 * np.linalg.norm(b) + 1e-9, n
    for w, m in (("W1", "M_W1"), ("W2", "M_W2")):
        # the update of the device's own gradient
        rows_, cols = d[w].shape
        nw, nm, x = rows.muon64(d[w], got.output("d" + w), np.zeros_like(d[w]), 1e-2, 0.95, True, 5, 0.01, max(1.0, rows_ / cols) ** 0.5)
        assert np.linalg.norm(got.output(w) - nw) <= 1e-4 * 1e-2 * max(1.0, rows_ / cols) ** 0.5 * np.linalg.norm(x) + 4 * 2.0 ** -24 * np.linalg.norm(nw)
        assert np.abs(got.output(m) - nm).max() <= 2 * 2.0 ** -24 * np.abs(nm).max()
    for _ in range(4):                                       # (from the third run on small programs are graphs)
        got.run()
    first = {n: got.output(n) for n in program.outputs}
    again = begin(DeviceExecutor(fuse_program(program) if fused else program), d)
    for _ in range(5):
        again.run()
    assert all(np.array_equal(again.output(n), first[n]) for n in program.outputs)

