"""fadamw against its definition: moments and codes to the bit, weights to a few roundings of U = 2^-24."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INV_MAX = np.float32(1 / 448)


@pytest.fixture(scope="module")
def env():
    import torch
    import __graft_entry__ as ge
    ge.load_package()
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return torch, DeviceBuiltins()


def padded(a, n=128):
    return np.concatenate([a, np.zeros(-len(a) % n, a.dtype)]).reshape(-1, n)


def codes_of(torch, x, never_zero):
    """x [blocks, 128] in float32 as e4m3 codes and scales, as the builtin defines them."""
    largest = np.abs(x).max(1)
    with np.errstate(all="ignore"):
        scale = np.where(largest < np.float32(2.0 ** -100), np.float32(0), largest * INV_MAX).astype(np.float32)
        y = np.where(scale[:, None] == 0, np.float32(0), x * np.where(scale == 0, np.float32(0), np.float32(1) / scale)[:, None])
    q = torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy().copy()
    if never_zero:
        q[(q == 0) & (x > 0) & (scale > 0)[:, None]] = 1
    return q, scale


def values_of(torch, q, scale):
    return torch.from_numpy(q).view(torch.float8_e4m3fn).float().numpy() * scale[:, None]


def expect(torch, w, g, m, v, step, lr, b1, b2, eps, decay, eight=None):
    """New weights in 64 bits and how far they may be off; moments (or codes and scales) to the bit."""
    f = np.float32
    b1, b2 = f(b1), f(b2)
    if eight:
        q1, s1, q2, s2 = eight
        m = values_of(torch, q1, s1)
        u = values_of(torch, q2, s2)
        with np.errstate(all="ignore"):
            v = u * u
        g = padded(g)
    with np.errstate(all="ignore"):
        m = m * b1 + g * (f(1) - b1)
        v = v * b2 + g * (f(1) - b2) * g
    n = len(w)
    m64, v64 = m.reshape(-1)[:n].astype(np.float64), v.reshape(-1)[:n].astype(np.float64)
    c1, c2 = 1 - float(b1) ** step, 1 - float(b2) ** step
    with np.errstate(all="ignore"):
        update = lr / c1 * m64 / (np.sqrt(v64 / c2) + float(f(eps)))
    keep = w.astype(np.float64) * (1 - lr * decay)
    # the factor of w: fp32's of 1 - lr * decay, twice rounded; the update: root, its factor, sum, quotient, rate (which has fp32's lr and
    # on the device the 4 roundings of a power) and the products; the difference
    off = U * (4 * np.abs(keep) + 16 * np.abs(update) + np.abs(keep - update))
    if not eight:
        return keep - update, off, m, v
    with np.errstate(all="ignore"):
        root = np.sqrt(v)
    return keep - update, off, codes_of(torch, m, False), codes_of(torch, root, True)


def make(torch, n, eight, seed=0, offset=0):
    rng = np.random.default_rng(n + seed)
    a = {"w": rng.standard_normal(n), "g": rng.standard_normal(n) * 1e-2 * np.exp(rng.standard_normal(n) * 3), "m": rng.standard_normal(n) * 1e-2,
         "v": (rng.standard_normal(n) * 1e-2) ** 2}
    a = {k: x.astype(np.float32) for k, x in a.items()}
    if n > 300:
        a["g"][130:290], a["m"][128:256], a["v"][128:256] = 0, 0, 0          # a block of nothing
        a["m"][256:300], a["v"][256:300] = 0, 0
    if eight:
        a["q1"], a["s1"] = codes_of(torch, padded(a.pop("m")), False)
        a["q2"], a["s2"] = codes_of(torch, np.sqrt(padded(a.pop("v"))), True)
    dev = {}
    for k, x in a.items():
        x = x.reshape(-1)[:n] if k[0] == "q" else x
        t = torch.zeros(len(x) + offset, dtype=torch.uint8 if k[0] == "q" else torch.float32, device="cuda")[offset:]
        t.copy_(torch.from_numpy(np.ascontiguousarray(x)))
        dev[k] = t
    return a, dev


def check(torch, host, dev, n, eight, step, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.01):
    if not eight:
        w, off, m, v = expect(torch, host["w"], host["g"], host["m"], host["v"], step, lr, b1, b2, eps, decay)
        assert np.array_equal(dev["m"].cpu().numpy(), m, equal_nan=True) and np.array_equal(dev["v"].cpu().numpy(), v, equal_nan=True)
    else:
        w, off, (q1, s1), (q2, s2) = expect(torch, host["w"], host["g"], None, None, step, lr, b1, b2, eps, decay,
                                            tuple(host[k] for k in ("q1", "s1", "q2", "s2")))
        assert np.array_equal(dev["s1"].cpu().numpy(), s1, equal_nan=True) and np.array_equal(dev["s2"].cpu().numpy(), s2, equal_nan=True)
        assert np.array_equal(dev["q1"].cpu().numpy(), q1.reshape(-1)[:n]) and np.array_equal(dev["q2"].cpu().numpy(), q2.reshape(-1)[:n])
    got = dev["w"].cpu().numpy().astype(np.float64)
    fine = np.isfinite(w)
    assert np.array_equal(fine, np.isfinite(got))
    assert (np.abs(got - w)[fine] <= 1.000001 * off[fine] + 1e-40).all(), float((np.abs(got - w)[fine] - off[fine]).max())


def step_of(d, devs, eight, **k):
    col = lambda name: [x[name] for x in devs]  # noqa: E731
    moments = [col("q1"), col("q2"), col("s1"), col("s2")] if eight else [col("m"), col("v")]
    d.fadamw(col("w"), col("g"), *moments, **k)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 31, 127, 128, 129, 255, 1000, 1024, 4097, 100003, 1 << 20])
def test_one_tensor(env, n, eight):
    torch, d = env
    for offset, step in ((0, 1), (0, 1000), (1, 7), (2, 7), (3, 7)) if n in (3, 129, 4097) else ((0, 3),):
        host, dev = make(torch, n, eight, offset=offset)
        step_of(d, [dev], eight, step=step, lr=1e-3)
        check(torch, host, dev, n, eight, step)


@pytest.mark.parametrize("eight", [False, True])
def test_many_tensors_share_a_step(env, eight):
    torch, d = env
    rng = np.random.default_rng(3)
    sizes = [int(x) for x in np.exp(rng.uniform(0, 11, 700))] + [0, 300000, 0]
    pairs = [make(torch, n, eight, seed=i) for i, n in enumerate(sizes)]
    decays = [float(i % 3) * 0.1 for i in range(len(sizes))]
    step_of(d, [p[1] for p in pairs], eight, step=12, lr=3e-3, beta1=0.8, beta2=0.95, eps=1e-6, weight_decay=decays)
    for (host, dev), n, decay in zip(pairs, sizes, decays):
        if n:
            check(torch, host, dev, n, eight, 12, 3e-3, 0.8, 0.95, 1e-6, decay)


@pytest.mark.parametrize("eight", [False, True])
def test_nothing_beyond_a_tensor_is_touched(env, eight):
    torch, d = env
    n, room = 1000, 64
    host, dev = make(torch, n, eight)
    around = {}
    for k, t in dev.items():
        buf = torch.full((len(t) + 2 * room,), 77, dtype=t.dtype, device="cuda")
        buf[room:-room] = t
        around[k], dev[k] = buf, buf[room:-room]
    step_of(d, [dev], eight, step=3, lr=1e-3)
    check(torch, host, dev, n, eight, 3)
    assert all((b[:room] == 77).all() and (b[-room:] == 77).all() for b in around.values())


@pytest.mark.parametrize("eight", [False, True])
def test_a_schedule_on_the_device_is_read_at_each_replay(env, eight):
    torch, d = env
    n = 3001
    host, dev = make(torch, n, eight)
    again = {k: v.clone() for k, v in dev.items()}
    schedule = torch.tensor([0.0, 2e-3], device="cuda")
    one = torch.tensor([1.0, 0.0], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d.fadd(schedule, 1.0, one, 1.0, schedule)
        step_of(d, [dev], eight, schedule=schedule)
    for step in range(1, 6):
        before = {k: v.clone().cpu().numpy() for k, v in dev.items()}
        if eight:
            for k in ("q1", "q2"):
                before[k] = padded(before[k])
        graph.replay()
        check(torch, before, dev, n, eight, step, lr=2e-3)
        step_of(d, [again], eight, step=step, lr=2e-3)
        moments = ("q1", "q2", "s1", "s2") if eight else ("m", "v")
        assert all(torch.equal(dev[k], again[k]) for k in moments)
    assert schedule.tolist() == [5.0, float(np.float32(2e-3))]


def test_values_at_the_edges(env):
    torch, d = env
    n = 512
    for eight in (False, True):
        host, dev = make(torch, n, eight)
        g = host["g"]
        g[:128] = 1e-36                                      # below the least scale, in squares below everything
        g[130], g[300], g[301] = np.nan, np.inf, -np.inf
        g[384:] = 0
        if eight:
            for k in ("q1", "s1", "q2", "s2"):
                host[k][0] = 0
                host[k][3] = 0
        else:
            for k in "mv":
                host[k][:128], host[k][384:] = 0, 0
        for k in host:
            dev[k].copy_(torch.from_numpy(np.ascontiguousarray(host[k].reshape(-1)[:len(dev[k])])))
        step_of(d, [dev], eight, step=1, lr=1e-3)
        if not eight:
            check(torch, host, dev, n, eight, 1)
            continue
        # a gradient that is no number spoils its block's moments, and no other
        assert not dev["s1"][0] and not dev["q1"][:128].any() and not dev["s2"][3] and not dev["q2"][384:].any()
        assert torch.isnan(dev["s1"][1]) and not torch.isfinite(dev["s1"][2])
        w = dev["w"].cpu()
        assert torch.isnan(w[130]) and torch.isfinite(w[:128]).all() and torch.isfinite(w[384:]).all()
        assert torch.isfinite(w[128:256]).sum() == 127 and torch.isfinite(w[256:384]).sum() >= 126
    # eps 0, nothing seen: 0 / 0, as the formula has it; betas of 0: the step is lr * sign
    host, dev = make(torch, 64, False)
    dev["g"].zero_(), dev["m"].zero_(), dev["v"].zero_()
    step_of(d, [dev], False, step=1, lr=1e-3, eps=0.0)
    assert torch.isnan(dev["w"]).all()
    host, dev = make(torch, 64, False)
    step_of(d, [dev], False, step=1, lr=1e-3, beta1=0.0, beta2=0.0, eps=0.0, weight_decay=0.0)
    want = torch.from_numpy(host["w"]).double() - 1e-3 * torch.sign(torch.from_numpy(host["g"])).double()
    assert (dev["w"].cpu().double() - want).abs().max() <= 8 * U * host["w"].__abs__().max() + 16 * U * 1e-3


def test_second_moments_in_8_bits_never_vanish_beside_their_first(env):
    # an element far below its block's largest keeps a divisor: without one the step after a gradient of zero would be m / eps
    torch, d = env
    n = 128
    dev = {"w": torch.zeros(n, device="cuda"), "g": torch.full((n,), 1e-6, device="cuda"), "q1": torch.zeros(n, dtype=torch.uint8, device="cuda"),
           "q2": torch.zeros(n, dtype=torch.uint8, device="cuda"), "s1": torch.zeros(1, device="cuda"), "s2": torch.zeros(1, device="cuda")}
    dev["g"][0] = 10.0
    for step in range(1, 20):
        step_of(d, [dev], True, step=step, lr=1e-3, weight_decay=0.0)
        dev["g"].zero_()
        assert dev["q2"].min() >= 1
    assert dev["w"].abs().max() < 20 * 1e-3 * math.sqrt(20)


def test_steps_on_two_streams(env):
    torch, d = env
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    pairs = [[make(torch, 5000, False, seed=i) for i in range(3)] for _ in streams]
    torch.cuda.synchronize()
    for s, p in zip(streams, pairs):
        with torch.cuda.stream(s):
            step_of(d, [x[1] for x in p], False, step=2, lr=1e-3)
    torch.cuda.synchronize()
    for p in pairs:
        for host, dev in p:
            check(torch, host, dev, 5000, False, 2)
