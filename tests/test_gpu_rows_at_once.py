"""Layer norm, log probabilities and AdamW called by several host threads at once, each on a stream of its own, and calls at the edge of what is allowed."""
import ctypes
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import __graft_entry__ as ge
    ge.load_package()
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return torch, DeviceBuiltins()


def step(torch, d, seed):
    """Everything on rows and weights once, on inputs of its own; the results."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, classes = 200 + 37 * seed, 600 + 41 * seed, 1500 + seed
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x, gamma, beta, g = rand(rows, cols), rand(cols), rand(cols), rand(rows, cols)
    logits, ids = rand(rows, classes), torch.randint(-1, classes, (rows,), device="cuda", generator=gen)
    new = lambda *s: torch.empty(*s, device="cuda")
    out, mean, rstd, dx, dgamma, dbeta = new(rows, cols), new(rows), new(rows), new(rows, cols), new(cols), new(cols)
    lp, ent, lse, top_lp, dl = new(rows), new(rows), new(rows), new(rows, 9), new(rows, classes)
    top = torch.empty(rows, 9, dtype=torch.int64, device="cuda")
    w, m, v = gamma.clone(), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    d.flayernorm(x, gamma, beta, 1e-5, out, mean, rstd)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx, dgamma, dbeta)
    d.flogprob(logits, ids, lp, ent, lse, top, top_lp)
    d.flogprob_grad(logits, ids, lse, ent, lp, ent, dl)
    d.fadamw([w], [dgamma], [m], [v], step=1, lr=1e-2)
    return [out, mean, rstd, dx, dgamma, dbeta, lp, ent, lse, top, top_lp, dl, w, m, v]


def test_threads_with_streams_of_their_own(env):
    torch, d = env
    n = 4
    alone = [step(torch, d, i) for i in range(n)]
    torch.cuda.synchronize()
    got, errors = [None] * n, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = step(torch, d, i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                               # (an assertion in a thread would be lost)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_alternatives_of_two_widths_are_refused(env):
    torch, d = env
    x, ids, lp = torch.randn(6, 40, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda"), torch.empty(6, device="cuda")
    for a, b in ((0, 5), (5, 0), (4, 5)):
        with pytest.raises(ValueError):
            d.flogprob(x, ids, lp, None, None, torch.empty(6, a, dtype=torch.int64, device="cuda"), torch.empty(6, b, device="cuda"))


def test_one_gradient_for_two_tensors_and_moments_of_both_kinds_in_a_call(env):
    torch, d = env
    from polarai_framework_b200.capi import AdamwOptions, AdamwTensor
    n = 1000
    g = torch.randn(n, device="cuda")

    def state():
        return {"w": torch.linspace(-1, 1, n, device="cuda"), "m": torch.zeros(n, device="cuda"), "v": torch.zeros(n, device="cuda"),
                "q1": torch.zeros(n, dtype=torch.uint8, device="cuda"), "q2": torch.zeros(n, dtype=torch.uint8, device="cuda"),
                "s1": torch.zeros(8, device="cuda"), "s2": torch.zeros(8, device="cuda")}
    one, both = [state(), state()], [state(), state()]
    decay = np.float32(0.25)
    d.fadamw([one[0]["w"]], [g], [one[0]["m"]], [one[0]["v"]], step=1, lr=1e-2, weight_decay=decay)
    d.fadamw([one[1]["w"]], [g], [one[1]["q1"]], [one[1]["q2"]], [one[1]["s1"]], [one[1]["s2"]], step=1, lr=1e-2, weight_decay=decay)
    a, b = both
    tensors = (AdamwTensor * 2)(
        AdamwTensor(b["w"].data_ptr(), g.data_ptr(), b["q1"].data_ptr(), b["q2"].data_ptr(), b["s1"].data_ptr(), b["s2"].data_ptr(), n, float(decay)),
        AdamwTensor(a["w"].data_ptr(), g.data_ptr(), a["m"].data_ptr(), a["v"].data_ptr(), None, None, n, float(decay)))
    options = AdamwOptions(1e-2, 0.9, 0.999, 1e-8, 1, None)
    d.lib.call("polar_b200_fadamw", tensors, 2, ctypes.byref(options), torch.cuda.current_stream().cuda_stream)
    for x, y in zip(one, both):
        assert all(torch.equal(x[k], y[k]) for k in x)
