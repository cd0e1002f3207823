"""The oracle's updates with moments in 8 bits and its alternatives: against torch's e4m3 on the host, and the GPU's programs against it."""
import numpy as np
import pytest
import torch

import __graft_entry__ as ge

ge.load_package()
from oracle import rows_oracle as rows  # noqa: E402
from oracle.program_executor import OracleExecutor  # noqa: E402
from polarai_framework_b200.program import Program, norm_classifier_program  # noqa: E402
from test_norm_classifier import begin, data  # noqa: E402

U = 2.0 ** -24


def test_codes_are_torchs():
    codes = np.arange(256, dtype=np.uint8)
    values = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(rows.from_e4m3(codes), values, equal_nan=True)
    rng = np.random.default_rng(0)
    between = np.sort(values[np.isfinite(values)])
    y = np.concatenate([values[np.isfinite(values)], (between[1:] + between[:-1]) / 2, rng.standard_normal(5000) * np.exp(rng.standard_normal(5000) * 4),
                        [0.0, -0.0, 448.0, 463.9, -448.0, 2.0 ** -10, 1.5 * 2.0 ** -10, np.nan]]).astype(np.float32)
    y = y[np.isnan(y) | (np.abs(y) < 464)]                   # (beyond, torch gives NaN where the builtin saturates)
    assert np.array_equal(rows.to_e4m3(y) & 0x7f, torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy() & 0x7f)
    assert rows.to_e4m3(np.float32([500, -1e30, np.inf])).tolist() == [0x7e, 0xfe, 0x7e]


def test_a_program_with_moments_in_8_bits_on_the_oracle(oracle):
    # the first step begins with zeros: the codes hold (1 - beta1) g to half a step of e4m3, 2^-4 of it, or of its block's least
    shape = (9, 8, 33, 5)
    d = data(*shape)
    ex, wide = (begin(OracleExecutor(norm_classifier_program(*shape, state_bits=b), oracle), d) for b in (8, 32))
    ex.run(), wide.run()
    for w in ("W1", "W2", "gamma", "beta"):
        n, m = ex.t[w].size, wide.t["m_" + w].ravel()
        scale = np.repeat(ex.t["ms_" + w], 128)[:n]
        got = rows.from_e4m3(ex.t["m_" + w].view(np.uint8)[:n]) * scale
        assert (np.abs(got - m) <= 2.0 ** -4 * np.abs(m) * (1 + 4 * U) + 2.0 ** -10 * scale).all()
        # the step itself is made of the moments before they are rounded; both take the root in another place
        assert np.abs(ex.t[w].astype(np.float64) - wide.t[w]).max() <= 8 * U * (np.abs(wide.t[w]).max() + 1e-2)
    for _ in range(3):
        ex.run()
    assert ex.t["schedule"][0] == 4 and all(np.isfinite(ex.t[w]).all() for w in ("W1", "W2", "gamma", "beta"))


def alternatives(rows_, classes, top):
    p = Program("alternatives")
    p.tensor("x", rows_, classes), p.tensor("ids", rows_)
    for n in ("lp", "ent", "lse"):
        p.tensor(n, rows_)
    p.tensor("tops", rows_, top), p.tensor("toplp", rows_, top)
    p.inputs, p.outputs = ["x", "ids"], ["lp", "ent", "lse", "tops", "toplp"]
    p.op("flogprob_top", "x", "ids", "lp", "ent", "lse", "tops", "toplp")
    rng = np.random.default_rng(classes)
    x = (rng.standard_normal((rows_, classes)) * 2).astype(np.float32)
    x[:, ::7] = x[:, :1]                                     # ties
    return p, {"x": x, "ids": rng.integers(-1, classes, rows_).astype(np.float32)}


def test_alternatives_in_a_program_on_the_oracle(oracle):
    p, given = alternatives(6, 40, 9)
    ex = OracleExecutor(p, oracle)
    ex.set_inputs(**given)
    ex.run()
    x = torch.from_numpy(given["x"]).double()
    lp, at = torch.sort(torch.log_softmax(x, 1), dim=1, descending=True, stable=True)
    assert np.array_equal(ex.t["tops"], at[:, :9].numpy().astype(np.float32))
    assert np.abs(ex.t["toplp"] - lp[:, :9].numpy()).max() <= 4 * U * np.abs(lp[:, :9].numpy()).max()


# ---- on the GPU

@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(33, 20, 36, 7), (64, 31, 1000, 300)])
def test_steps_with_moments_in_8_bits_against_the_oracle(shape):
    # each of several steps of the program: the moments to the bit, from the device's own gradients and the state before
    from polarai_framework_b200.program import DeviceExecutor
    ex = begin(DeviceExecutor(norm_classifier_program(*shape, state_bits=8)), data(*shape), lr=1e-3)
    names = ("W1", "W2", "gamma", "beta")
    for step in range(1, 5):
        before = {n: ex.output(n) for w in names for n in (w, "m_" + w, "ms_" + w, "v_" + w, "vs_" + w)}
        ex.run()
        for w in names:
            n, g, decay = before[w].size, ex.output("d" + w), 0.01 if w[0] == "W" else 0.0
            codes = lambda a: a.view(np.uint8)[:n]  # noqa: E731
            new, q1, s1, q2, s2 = rows.fadamw8(before[w], g, codes(before["m_" + w]), before["ms_" + w], codes(before["v_" + w]), before["vs_" + w],
                                               step, 1e-3, 0.9, 0.999, 1e-8, decay)
            assert np.array_equal(ex.output("ms_" + w), s1) and np.array_equal(ex.output("vs_" + w), s2)
            assert np.array_equal(codes(ex.output("m_" + w)), q1) and np.array_equal(codes(ex.output("v_" + w)), q2)
            # as in test_gpu_adamw.py: 4 roundings of the weight, 16 of the update, one of their difference
            update = np.abs(new.astype(np.float64) - before[w]) + 1e-3 * decay * np.abs(before[w])
            off = U * (5 * np.abs(before[w]) + 18 * update)
            assert (np.abs(ex.output(w).astype(np.float64) - new) <= off + U * np.abs(new) + 1e-40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows_,classes,top", [(6, 40, 9), (300, 700, 32), (1000, 100, 5), (3, 20000, 20)])
def test_alternatives_in_a_program_against_the_oracle(oracle, rows_, classes, top):
    from polarai_framework_b200.program import DeviceExecutor
    p, given = alternatives(rows_, classes, top)
    ex, want = DeviceExecutor(p), OracleExecutor(p, oracle)
    for e in (ex, want):
        e.set_inputs(**given)
        e.run()
    assert np.array_equal(ex.output("tops"), want.t["tops"])
    # exponentials off by 2 |d| U + 4 U with |d| below 30, sums of classes / 32 + 40 additions at most, a logarithm and a few roundings of
    # values below 30; the entropy multiplies the exponentials' errors with deviations below 30
    off = U * (classes / 32 + 40 + 64 + 4 * 30)
    for n in ("lp", "lse", "toplp"):
        assert np.abs(ex.output(n).astype(np.float64) - want.t[n]).max() <= off
    assert np.abs(ex.output("ent").astype(np.float64) - want.t["ent"]).max() <= 30 * off
