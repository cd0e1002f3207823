"""A training step made of the builtins on rows and weights - matmul, layer norm, sigmoid, matmul, log probability, their gradients,
AdamW - as one program: on the oracle against differences, on the GPU against the oracle."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from oracle import rows_oracle as rows  # noqa: E402
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.program import Program, fuse_program, norm_classifier_program, results_of  # noqa: E402


def data(batch, n_in, n_hidden, classes, seed=0, padded=True):
    rng = np.random.default_rng(seed)
    labels = rng.integers(0, classes, batch).astype(np.float32)
    if padded and batch > 4:
        labels[::5] = -1.0
    return {"X": rng.standard_normal((batch, n_in)).astype(np.float32), "labels": labels,
            "W1": (rng.standard_normal((n_in, n_hidden)) / np.sqrt(n_in)).astype(np.float32),
            "W2": (rng.standard_normal((n_hidden, classes)) / np.sqrt(n_hidden)).astype(np.float32),
            "gamma": (1 + 0.1 * rng.standard_normal(n_hidden)).astype(np.float32), "beta": (0.1 * rng.standard_normal(n_hidden)).astype(np.float32)}


def begin(ex, inputs, lr=1e-2):
    ex.set_inputs(**inputs, schedule=np.array([0, lr], np.float32), tick=np.array([1, 0], np.float32))
    zeros = [n for n in ex.program.inputs if n not in inputs and n not in ("schedule", "tick")]
    if hasattr(ex, "set_zeros"):
        ex.set_zeros(*zeros)
    return ex


def forward64(d):
    f = {k: v.astype(np.float64) for k, v in d.items()}
    z = f["X"] @ f["W1"]
    dev = z - z.mean(1, keepdims=True)
    n = dev / np.sqrt((dev ** 2).mean(1, keepdims=True) + np.float64(np.float32(1e-5))) * f["gamma"] + f["beta"]
    h = 1 / (1 + np.exp(-n))
    l = h @ f["W2"]
    l = l - l.max(1, keepdims=True)
    l = l - np.log(np.exp(l).sum(1, keepdims=True))
    ids = d["labels"].astype(int)
    return -np.where(ids >= 0, l[np.arange(len(ids)), np.maximum(ids, 0)], 0.0).mean()


def test_gradients_of_the_step_against_differences(oracle):
    d = data(7, 5, 6, 4)
    ex = begin(OracleExecutor(norm_classifier_program(7, 5, 6, 4), oracle), d)
    ex.run()
    rng = np.random.default_rng(1)
    for name in ("W1", "W2", "gamma", "beta"):
        grad = ex.t["d" + name]
        for _ in range(8):
            at = tuple(rng.integers(0, s) for s in grad.shape)
            shifted = []
            for step in (1e-3, -1e-3):
                e = {k: v.astype(np.float64) for k, v in d.items()}
                e[name][at] += step
                e["labels"] = d["labels"]
                shifted.append(forward64(e))
            # differences: third derivatives (below 10) times 1.7e-7; the gradient: fp32 sums of a few terms below 1
            assert abs((shifted[0] - shifted[1]) / 2e-3 - grad[at]) < 5e-6


def test_the_fused_form_is_the_same_program(oracle):
    d = data(9, 8, 12, 5)
    plain = norm_classifier_program(9, 8, 12, 5)
    fused = fuse_program(plain)
    names = [k for k, _ in fused.ops]
    assert "fdense_grad" in names and "fsigmoid_grad" not in names and len(fused.ops) == len(plain.ops) - 4
    a, b = (begin(OracleExecutor(p, oracle), d) for p in (plain, fused))
    for _ in range(3):
        a.run(), b.run()
    assert all(np.array_equal(a.t[n], b.t[n]) for n in plain.outputs)


def test_a_product_does_not_move_past_the_update_of_its_operand():
    p = Program("between")
    for n in ("X", "W", "Z", "H", "g", "m", "v"):
        p.tensor(n, 4, 4)
    p.tensor("schedule", 2)
    p.inputs, p.outputs = ["X", "W", "g", "m", "v", "schedule"], ["H"]
    p.op("fmatmul_f_f", "X", "W", "Z")
    p.op("fadamw", "g", "schedule", 0.9, 0.999, 1e-8, 0.0, "W", "m", "v")
    p.op("fsigmoid", "Z", "H")
    assert [k for k, _ in fuse_program(p).ops] == ["fmatmul_f_f", "fadamw", "fsigmoid"]
    assert results_of(*p.ops[1]) == ["W", "m", "v"] and results_of(*p.ops[0]) == ["Z"]


def test_two_ranks_share_a_batch(oracle):
    # the sum of the gradients of two halves of a batch, as ALLREDUCE gives it to both: the same update as of the whole
    d = data(10, 6, 8, 4)
    whole = begin(OracleExecutor(norm_classifier_program(10, 6, 8, 4), oracle), d)
    whole.run()
    halves, sums = [], []
    for i in range(2):
        part = {k: (v[5 * i:5 * i + 5] if k in ("X", "labels") else v) for k, v in d.items()}
        halves.append(begin(OracleExecutor(norm_classifier_program(5, 6, 8, 4, samples=10), oracle), part))
    for ex in halves:
        ex.run()
    for name in ("W1", "W2", "gamma", "beta"):
        sums.append(np.abs(halves[0].t["d" + name] + halves[1].t["d" + name] - whole.t["d" + name]).max())
    assert max(sums) < 16 * 2.0 ** -24                       # sums of ten terms below 1, each rounded once more


# ---- on the GPU

SHAPES = [(33, 20, 36, 7), (257, 784, 512, 10), (64, 31, 1000, 300)]


def relative(got, want):
    return float(np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want))


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_the_step_on_the_gpu_against_the_oracle(oracle, shape, fused):
    from polarai_framework_b200.program import DeviceExecutor
    d = data(*shape)
    prog = norm_classifier_program(*shape)
    ex = begin(DeviceExecutor(fuse_program(prog) if fused else prog), d, lr=1e-3)
    want = begin(OracleExecutor(prog, oracle), d, lr=1e-3)
    ex.run(), want.run()
    # products of up to n_in (784) and n_hidden (1000) terms, at up to 1e-8 of the result per term and 1e-6 at least; four layers of them,
    # the norm and the sigmoid in between, each of which passes an error on with a factor of a few: 1e-4 of the norm of a result
    for n in ("logp", "entropy", "dW1", "dW2", "dgamma", "dbeta"):
        assert relative(ex.output(n), want.t[n]) < 1e-4, n
    # a first step moves a weight by lr times sign(g) where g is not lost in eps: compare what the step was made of instead
    for w in ("W1", "W2", "gamma", "beta"):
        g, decay = ex.output("d" + w), 0.01 if w[0] == "W" else 0.0
        new, m, v = rows.fadamw(d[w], g, np.zeros_like(g), np.zeros_like(g), 1, 1e-3, 0.9, 0.999, 1e-8, decay)
        assert np.array_equal(ex.output("m_" + w), m) and np.array_equal(ex.output("v_" + w), v)
        step = np.abs(new - d[w].astype(np.float64)) + np.abs(d[w])
        assert (np.abs(ex.output(w).astype(np.float64) - new) <= 24 * 2.0 ** -24 * step + 1e-40).all()
    assert ex.output("schedule").tolist() == [1.0, float(np.float32(1e-3))]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_replayed_as_a_graph_are_the_steps_launched_one_by_one(bits):
    import torch
    from polarai_framework_b200.capi import lib
    from polarai_framework_b200.program import DeviceExecutor
    shape = (100, 40, 260, 11)
    d = data(*shape)
    prog = fuse_program(norm_classifier_program(*shape, state_bits=bits))
    ex, single = begin(DeviceExecutor(prog), d), begin(DeviceExecutor(prog), d)
    # the four updates are one launch: of the program's ops all but those, one chain for the schedule among them
    steps = lib().cdll.polar_b200_program_steps(ex._only)
    assert steps == len([o for o in prog.ops if o[0] not in ("ALLREDUCE", "fadamw", "fadamw8")]) + 1
    eager = torch.cuda.CUDAGraph()                           # the other one inside a capture of the caller's, replayed
    with torch.cuda.graph(eager):
        single.run()
    begin(single, d)
    for _ in range(6):
        ex.run()                                             # from the third run on a graph of its own
        eager.replay()
    torch.cuda.synchronize()
    for n in prog.inputs + prog.outputs:
        assert torch.equal(ex.t[n].view(torch.int32), single.t[n].view(torch.int32)), n
    assert ex.output("schedule")[0] == 6.0
    assert np.isfinite(ex.output("logp")).all() and (ex.output("logp")[::5] == 0).all()


@pytest.mark.gpu
def test_updates_that_depend_on_each_other_stay_apart():
    import torch
    from polarai_framework_b200.capi import lib
    from polarai_framework_b200.program import DeviceExecutor
    p = Program("twice")
    for n in ("W", "m", "v", "g", "U", "mu", "vu"):
        p.tensor(n, 300)
    p.tensor("schedule", 2)
    p.inputs, p.outputs = list(p.tensors), ["W", "U"]
    p.op("fadamw", "g", "schedule", 0.9, 0.999, 1e-8, 0.0, "W", "m", "v")
    p.op("fadamw", "g", "schedule", 0.9, 0.999, 1e-8, 0.0, "W", "m", "v")        # the same weights again
    p.op("fadamw", "W", "schedule", 0.9, 0.999, 1e-8, 0.0, "U", "mu", "vu")      # with what the others write as its gradient
    p.op("fadamw", "g", "schedule", 0.8, 0.999, 1e-8, 0.0, "g", "m", "v")        # other betas
    ex = DeviceExecutor(p)
    assert lib().cdll.polar_b200_program_steps(ex._only) == 4
    rng = np.random.default_rng(0)
    w, g, u = (rng.standard_normal(300).astype(np.float32) for _ in range(3))
    z = np.zeros(300, np.float32)
    ex.set_inputs(W=w, g=g, U=u, m=z, v=z, mu=z, vu=z, schedule=np.array([3, 1e-2], np.float32))
    ex.run()
    torch.cuda.synchronize()
    a = rows.fadamw(w, g, z, z, 3, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    a = rows.fadamw(a[0], g, a[1], a[2], 3, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    assert np.abs(ex.output("W") - a[0]).max() <= 32 * 2.0 ** -24 * np.abs(w).max()
    assert np.abs(ex.output("mu") - np.float32(0.1) * a[0]).max() <= 8 * 2.0 ** -24 * np.abs(w).max()


@pytest.mark.gpu
def test_every_name_gives_what_its_entry_point_gives():
    import torch
    from polarai_framework_b200.device_builtins import DeviceBuiltins, HostBuiltins
    from polarai_framework_b200.program import DeviceExecutor
    rows_, cols, top = 37, 50, 6
    rng = np.random.default_rng(2)
    p = Program("names")
    x = {"x": (rows_, cols), "gamma": (cols,), "beta": (cols,), "out": (rows_, cols), "mean": (rows_,), "rstd": (rows_,), "dout": (rows_, cols),
         "dx": (rows_, cols), "dgamma": (cols,), "dbeta": (cols,), "ids": (rows_,), "lp": (rows_,), "ent": (rows_,), "lse": (rows_,),
         "tops": (rows_, top), "toplp": (rows_, top), "g": (rows_,), "gh": (rows_,), "dl": (rows_, cols), "dl2": (rows_, cols)}
    for n, s in x.items():
        p.tensor(n, *s)
    p.inputs = ["x", "gamma", "beta", "dout", "ids", "g", "gh"]
    p.op("flayernorm", "x", "gamma", "beta", 1e-5, "out", "mean", "rstd")
    p.op("flayernorm_grad", "dout", "x", "gamma", "mean", "rstd", "dx", "dgamma", "dbeta")
    p.op("flogprob_top", "out", "ids", "lp", "ent", "lse", "tops", "toplp")
    p.op("flogprob_grad", "out", "ids", "lse", "g", "dl")
    p.op("flogprob_grad", "out", "ids", "lse", "ent", "g", "gh", "dl2")
    p.outputs = list(x)
    ex = DeviceExecutor(p)
    given = {n: rng.standard_normal(x[n]).astype(np.float32) for n in p.inputs}
    given["ids"] = rng.integers(-1, cols, rows_).astype(np.float32)
    ex.set_inputs(**given)
    ex.run()
    h = HostBuiltins()
    out, mean, rstd = h.flayernorm(given["x"], given["gamma"], given["beta"], 1e-5)
    same = lambda n, v: np.array_equal(ex.output(n), v)  # noqa: E731
    assert same("out", out) and same("mean", mean) and same("rstd", rstd)
    assert all(same(n, v) for n, v in zip(("dx", "dgamma", "dbeta"), h.flayernorm_grad(given["dout"], given["x"], given["gamma"], mean, rstd)))
    lp, ent, lse, tops, toplp = h.flogprob(out, given["ids"], top)
    assert same("lp", lp) and same("ent", ent) and same("lse", lse) and same("tops", tops.astype(np.float32)) and same("toplp", toplp)
    assert same("dl", h.flogprob_grad(out, given["ids"], lse, None, given["g"], None))
    assert same("dl2", h.flogprob_grad(out, given["ids"], lse, ent, given["g"], given["gh"]))
    for got, want in zip((lp, ent, lse, tops, toplp), rows.flogprob(out, given["ids"], top)):
        assert np.allclose(got, want, rtol=1e-5, atol=1e-5)
    w = rng.standard_normal(100).astype(np.float32)
    assert np.abs(h.fadamw(w, w, w, w * w, 5, 1e-3, 0.9, 0.99, 1e-8, 0.1)[0] - rows.fadamw(w, w, w, w * w, 5, 1e-3, 0.9, 0.99, 1e-8, 0.1)[0]).max() < 1e-6
    assert DeviceBuiltins().device_status() == 0 and torch.cuda.is_available()
