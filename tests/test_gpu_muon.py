"""Orthogonalised momentum against the formula in 64 bits.

Tolerance of the update, in the Frobenius norm and relative: a product holds 22 bits of its operands (2^-21 of a sum's terms in all) and its
sums are cut towards zero up to 24 times between two rounded additions, each time by less than 2^-23: 3.4e-6 of the terms' magnitude, whose
cuts all have one direction.  15 products make 5.1e-5, and a round changes a relative error by |s p'(s) / p(s)|, which is 1 for small singular
values s and below 2 where they have settled: 1e-4."""
import ctypes
import math

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from oracle import rows_oracle as rows  # noqa: E402

pytestmark = pytest.mark.gpu
U, CLOSE = 2.0 ** -24, 1e-4
A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def f(v):
    return float(np.float32(v))


def reference(w, g, m, lr, momentum=0.95, nesterov=True, steps=5, weight_decay=0.0, scale=None, coefficients=(A, B, C)):
    """(weights, momentum, update) in 64 bits, of matrices [..., rows, cols]."""
    a, b, c = (f(v) for v in coefficients)
    m = f(momentum) * m.double() + g.double()
    u = g.double() + f(momentum) * m if nesterov else m
    size = u.pow(2).sum((-2, -1), keepdim=True).sqrt()
    x = torch.where(size > 0, u / size, u)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    x = x.mT if tall else x
    scale = max(1.0, w.shape[-2] / w.shape[-1]) ** 0.5 if scale is None else scale
    return w.double() * (1 - f(lr) * f(weight_decay)) - f(lr) * f(scale) * x, m, x


def make(shape, seed=0, rank=None, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(1000 * seed + sum(shape))
    def one(scale):
        n = math.prod(shape)
        t = torch.empty(n + 8, device="cuda")[offset:offset + n].view(shape)
        return t.copy_(torch.randn(shape, device="cuda", generator=gen) * scale)
    w, g, m = one(0.02), one(1e-3), one(1e-2)
    if rank is not None:
        few = torch.randn((*shape[:-1], rank), device="cuda", generator=gen) @ torch.randn((*shape[:-2], rank, shape[-1]), device="cuda", generator=gen)
        g.copy_(few), m.copy_(few * 3)
    return w, g, m


def check(got_w, got_m, w, g, m, lr=0.5, close=CLOSE, **k):
    """The update that the new weights show, and the momentum to its rounding (a product and a sum as one operation)."""
    want_w, want_m, x = reference(w, g, m, lr, **k)
    scale = k.get("scale")
    scale = max(1.0, w.shape[-2] / w.shape[-1]) ** 0.5 if scale is None else scale
    # of the weights: their own rounding (three operations), and the update's share
    error = (got_w.double() - want_w).norm().item()
    assert error <= close * f(lr) * abs(scale) * x.norm().item() + 4 * U * want_w.norm().item(), (error, x.norm().item())
    assert ((got_m.double() - want_m).abs() <= 2 * U * want_m.abs() + 2 * U * (g.double().abs()) + 1e-44).all()


def step(d, ts, lr=0.5, **k):
    new = [(w.clone(), m.clone()) for w, _, m in ts]
    d.fmuon([n[0] for n in new], [t[1] for t in ts], [n[1] for n in new], lr=lr, **k)
    torch.cuda.synchronize()
    assert d.device_status() == 0
    return new


SHAPES = [(1, 1), (1, 2), (2, 1), (1, 1000), (1000, 1), (3, 5), (5, 3), (16, 16), (31, 33), (33, 31), (63, 65), (64, 64), (64, 128), (128, 64), (127, 129), (128, 128),
          (129, 127), (128, 1000), (1000, 128), (130, 70), (70, 130), (255, 257), (256, 256), (257, 255), (300, 1000), (1000, 300), (384, 640), (640, 384), (513, 511), (10, 4096),
          (4096, 10), (777, 1511), (1511, 777), (1024, 1024), (65, 5000), (5000, 65), (1280, 128), (2048, 512),
          # what one CTA holds ends at 128 x 256 and 64 x 512; far longer than wide beyond that
          (128, 300), (128, 512), (512, 128), (127, 513), (128, 2048), (2048, 128), (128, 2049), (100, 1000), (1000, 100), (64, 4096), (4096, 64), (64, 4097), (65, 2048),
          (33, 3000), (3000, 33), (32, 1025), (32, 8192), (8200, 32), (16, 2049), (16, 16384), (16384, 16), (17, 2000), (16, 20000), (5, 9000), (9000, 5), (1, 16384), (2, 2050),
          (48, 700), (700, 48), (96, 1030), (81, 1999),
          (128, 256), (256, 128), (128, 257), (257, 128), (129, 256), (64, 512), (512, 64), (64, 513), (65, 512), (65, 256), (512, 1), (1, 512), (17, 511), (100, 241)]


@pytest.mark.parametrize("shape", SHAPES)
def test_one_matrix(d, shape):
    w, g, m = make(shape)
    (nw, nm), = step(d, [(w, g, m)])
    check(nw, nm, w, g, m)


@pytest.mark.parametrize("shape", [(784, 4096), (4096, 784), (2048, 2048), (1100, 4500)])
def test_long_sums(d, shape):
    w, g, m = make(shape, 1, rank=8)
    g += 0.3 * torch.randn_like(g)
    (nw, nm), = step(d, [(w, g, m)])
    # half a step per cut on the average: 15 products of 24 * 2^-25 and 2^-22, twice
    check(nw, nm, w, g, m, close=3e-5)


@pytest.mark.parametrize("shape", [(40, 60), (200, 300), (300, 200), (1024, 512), (100, 2000)])
@pytest.mark.parametrize("rank", [1, 3])
def test_matrices_of_low_rank(d, shape, rank):
    # X has singular values of zero; what rounding leaves there (2^-22 of |X|, spread over all of them) grows by 3.4445^5 = 485: 1.2e-4, of which a
    # result of rank r has sqrt(r) as its norm
    w, g, m = make(shape, 2, rank=rank)
    (nw, nm), = step(d, [(w, g, m)])
    check(nw, nm, w, g, m, close=CLOSE + 485 * 2.0 ** -22)


def test_singular_values_come_together(d):
    w, g, m = make((300, 500), 3)
    (nw, _), = step(d, [(w, g, m)], lr=1.0, scale=1.0)
    s = torch.linalg.svdvals(w.double() - nw.double())
    assert 0.3 < s.min() and s.max() < 1.21                  # (the smallest of a random matrix need not have grown all the way)


@pytest.mark.parametrize("k", [{"nesterov": False}, {"momentum": 0.0}, {"steps": 1}, {"steps": 2}, {"steps": 3}, {"steps": 4}, {"steps": 8}, {"weight_decay": 0.1},
                               {"scale": 0.2}, {"scale": -1.0}, {"coefficients": (1.5, -0.5, 0.0)}, {"coefficients": (1.875, -1.25, 0.375)}])
@pytest.mark.parametrize("shape", [(100, 60), (90, 400), (1100, 90), (300, 500), (600, 300)])
def test_options(d, shape, k):
    w, g, m = make(shape, 4)
    (nw, nm), = step(d, [(w, g, m)], **k)
    check(nw, nm, w, g, m, **k)


def test_several_shapes_stacks_and_lists_of_options(d):
    shapes = [(64, 100), (3, 200, 130), (100, 64), (64, 100), (2, 2, 50, 50), (1, 7), (700, 300), (3, 200, 130), (0, 5), (4, 0, 3)]
    ts = [make(s, i) for i, s in enumerate(shapes)]
    decays, scales = [0.01 * i for i in range(len(ts))], [1.0 + 0.1 * i for i in range(len(ts))]
    for (nw, nm), t, decay, scale in zip(step(d, ts, weight_decay=decays, scale=scales), ts, decays, scales):
        if t[0].numel():
            check(nw, nm, *t, weight_decay=decay, scale=scale)


def test_more_shapes_than_a_launch_holds_and_more_matrices_than_a_table(d):
    ts = [make((20 + i, 300 + 3 * i), i) for i in range(19)]
    for (nw, nm), t in zip(step(d, ts), ts):
        check(nw, nm, *t)
    ts = [make((130 + i, 300 + 3 * i), i) for i in range(19)]
    for (nw, nm), t in zip(step(d, ts), ts):
        check(nw, nm, *t)
    ts = [make((8 + i % 3, 12), i) for i in range(850)]
    for (nw, nm), t in list(zip(step(d, ts), ts))[::37]:
        check(nw, nm, *t)
    ts = [make((130 + i % 2, 140), i) for i in range(410)]
    for (nw, nm), t in list(zip(step(d, ts), ts))[::31]:
        check(nw, nm, *t)


def test_narrow_and_small_matrices_beside_one_another(d):
    ts = [make(s, i) for i, s in enumerate([(128, 2000), (900, 100), (64, 700), (30, 8000), (60, 60), (16, 4000), (2, 5000), (128, 2000), (4, 120, 300)])]
    for (nw, nm), t in zip(step(d, ts), ts):
        check(nw, nm, *t)
    ts.append(make((300, 400), 20))
    for (nw, nm), t in zip(step(d, ts), ts):
        check(nw, nm, *t)
    ts = [make((100, 100 + i), i) for i in range(70)]        # more than the smaller table of small ones holds
    for (nw, nm), t in list(zip(step(d, ts), ts))[::9]:
        check(nw, nm, *t)


@pytest.mark.parametrize("steps", [5, 2])
def test_more_narrow_shapes_than_a_launch_holds(d, steps):
    # short sides from 1 to 128, each matrix longer than one CTA holds, and stacks of them
    ts = [make((1 + i * 127 // 69, 520 + 3 * i), i) for i in range(70)] + [make((600 + i, 9 + i), i) for i in range(3)] + [make((5, 33, 1111), 3), make((4, 128, 513), 4)]
    for (nw, nm), t in zip(step(d, ts, steps=steps), ts):
        check(nw, nm, *t, steps=steps)


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("shape", [(60, 64), (130, 257), (512, 300), (300, 512), (60, 2000), (2000, 60)])
def test_tensors_off_16_bytes(d, shape, offset):
    w, g, m = make(shape, 5, offset=offset)
    nw, nm = make(shape, 5, offset=offset)[::2]
    d.fmuon([nw], [g], [nm], lr=0.5)
    check(nw, nm, w, g, m)


@pytest.mark.parametrize("shape", [(50, 70), (300, 200), (200, 900), (50, 3000), (2000, 100)])
def test_zeros_stay_and_what_is_not_finite_stays_in_its_matrix(d, shape):
    ts = [make(shape, i) for i in range(4)]
    ts[0][1].zero_(), ts[0][2].zero_()
    ts[1][1].view(-1)[7] = math.nan
    ts[2][1].view(-1)[-3] = math.inf
    new = step(d, ts, weight_decay=0.5)
    assert torch.equal(new[0][0], ts[0][0] * (1 - 0.25)) and (new[0][1] == 0).all()
    for i in (1, 2):
        assert torch.isnan(new[i][0]).all()
        finite = torch.isfinite(ts[i][1])
        assert torch.isfinite(new[i][1][finite]).all()
    check(*new[3], *ts[3], weight_decay=0.5)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
@pytest.mark.parametrize("shape", [(60, 90), (200, 500), (30, 5000)])
def test_gradients_of_any_size(d, shape, scale):
    w, g, m = make(shape, 6)
    g, m = g * scale, m * scale
    (nw, nm), = step(d, [(w, g, m)])
    check(nw, nm, w, g, m)


def test_one_large_entry_among_tiny_ones(d):
    # singular values far apart: the small ones are 2^-20 of |X| and stay as the formula has them, to what 22 bits of the largest hold
    w, g, m = make((100, 120), 7)
    g *= 2.0 ** -20
    m.zero_()
    g[3, 5] = 1.0
    (nw, nm), = step(d, [(w, g, m)])
    check(nw, nm, w, g, m, close=CLOSE + 485 * 2.0 ** -22)


def test_same_bits_each_time_and_on_other_streams(d):
    ts = [make(s, 8) for s in ((200, 300), (64, 64), (1000, 200), (90, 2000))]
    first = step(d, ts)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    again = []
    for s in streams:
        new = [(w.clone(), m.clone()) for w, _, m in ts]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            d.fmuon([n[0] for n in new], [t[1] for t in ts], [n[1] for n in new], lr=0.5)
        again.append(new)
    torch.cuda.synchronize()
    for new in again:
        assert all(torch.equal(a, b) for x, y in zip(first, new) for a, b in zip(x, y))


@pytest.mark.parametrize("shapes", [[(60, 70)], [(300, 200), (64, 64)], [(784, 512), (512, 10)], [(100, 1000), (7, 3000)]])
def test_captured_with_a_schedule(d, shapes):
    ts = [make(s, 9) for s in shapes]
    schedule = torch.tensor([1.0, 0.25], device="cuda")
    new = [(w.clone(), m.clone()) for w, _, m in ts]
    call = lambda: d.fmuon([n[0] for n in new], [t[1] for t in ts], [n[1] for n in new], schedule=schedule, weight_decay=0.1)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n, t in zip(new, ts):
        n[0].copy_(t[0]), n[1].copy_(t[2])
    schedule[1] = 0.5
    graph.replay()
    torch.cuda.synchronize()
    for n, t in zip(new, ts):
        check(*n, *t, lr=0.5, weight_decay=0.1)
    eager = step(d, ts, lr=0.5, weight_decay=0.1)
    assert all(torch.equal(a, b) for x, y in zip(new, eager) for a, b in zip(x, y))


def test_two_graphs_and_an_eager_step_between_them(d):
    ts = [make((300, 200), 10), make((70, 60), 10)]
    sets = [[(w.clone(), m.clone()) for w, _, m in ts] for _ in range(2)]
    graphs = []
    for new in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            d.fmuon([n[0] for n in new], [t[1] for t in ts], [n[1] for n in new], lr=0.5)
        graphs.append(graph)
    eager = step(d, ts)
    graphs[0].replay(), graphs[1].replay()
    torch.cuda.synchronize()
    for new in sets:
        assert all(torch.equal(a, b) for x, y in zip(new, eager) for a, b in zip(x, y))


def test_a_step_in_several_groups(d):
    # more matrices than fit the workspace of one group
    ts = [make((4096, 4096), i) for i in range(11)]
    new = step(d, ts)
    for i in (0, 10):
        check(*new[i], *ts[i])


def test_a_gradient_may_serve_several_weights(d):
    w, g, m = make((100, 80), 11)
    v, n = w * 2, m.clone()
    a, b, ma, mb = w.clone(), v.clone(), m.clone(), n.clone()
    d.fmuon([a, b], [g, g], [ma, mb], lr=0.5)
    check(a, ma, w, g, m), check(b, mb, v, g, n)


def test_by_name_and_in_a_program_with_its_neighbours(d):
    from polarai_framework_b200.program import DeviceExecutor, Program
    p = Program("updates")
    shapes = {"U": (90, 200), "V": (200, 90), "S": (3, 40, 50)}
    for n, s in shapes.items():
        for k in ("", "d", "m"):
            p.tensor(k + n, *s)
    p.tensor("schedule", 2)
    p.inputs = [k + n for n in shapes for k in ("", "d", "m")] + ["schedule"]
    p.outputs = list(shapes)
    for n in shapes:
        p.op("fmuon", "d" + n, "schedule", 0.9, 1.0, 5.0, 0.01, 0.7, n, "m" + n)
    ex = DeviceExecutor(p)
    rng = np.random.default_rng(12)
    data = {n: rng.standard_normal(s).astype(np.float32) for n, s in p.tensors.items() if n != "schedule"}
    ex.set_inputs(**data, schedule=np.array([1, 0.5], np.float32))
    before = d.lib.launch_count()
    ex.run()
    shared = d.lib.launch_count() - before
    for n in shapes:
        w, g, m = (torch.from_numpy(data[k + n]).cuda() for k in ("", "d", "m"))
        check(ex.t[n], ex.t["m" + n], w, g, m, lr=0.5, momentum=0.9, weight_decay=0.01, scale=0.7)
    one = Program("one", dict(p.tensors), p.ops[:1], p.inputs, {}, ["U"])
    ex1 = DeviceExecutor(one)
    before = d.lib.launch_count()
    ex1.run()
    assert shared < 2 * (d.lib.launch_count() - before) + 20   # three in a row share their launches


@pytest.mark.parametrize("short", [False, True])
def test_steps_of_a_program_run_again_and_again_with_any_workspace(d, short):
    """Four steps one after another of a program of short launches, which becomes a graph on the way; with the library's own scratch where the program's is too small."""
    from polarai_framework_b200.capi import binding
    from polarai_framework_b200.program import DeviceExecutor, Program
    p = Program("updates")
    shapes = {"U": (90, 600), "V": (300, 200), "W": (300, 200), "S": (40, 50)}
    for n, s in shapes.items():
        for k in ("", "d", "m"):
            p.tensor(k + n, *s)
    p.tensor("schedule", 2)
    p.inputs = [k + n for n in shapes for k in ("", "d", "m")] + ["schedule"]
    p.outputs = list(shapes)
    rows = [["U", "V"], ["W"], ["S"]]
    p.tensor("T", 90, 90)
    for row in rows:
        for n in row:
            p.op("fmuon", "d" + n, "schedule", 0.9, 1.0, 5.0, 0.01, 0.7, n, "m" + n)
        p.op("fmatmul_f_t", "dU", "dU", "T")
    ex = DeviceExecutor(p)
    rng = np.random.default_rng(13)
    data = {n: rng.standard_normal(s).astype(np.float32) for n, s in p.tensors.items() if n not in ("schedule", "T")}
    ex.set_inputs(**data, schedule=np.array([1, 0.5], np.float32))
    eager = {n: tuple(torch.from_numpy(data[k + n]).cuda() for k in ("", "d", "m")) for n in shapes}
    native = binding()
    handle = None
    if short:                                              # enough for the first matrix alone
        need = native.workspace_bytes([(k, ctypes.addressof(a), n) for k, a, n in ex._compiled[:1]])
        assert need < ex._ws_bytes
        status, handle = native.create_program([(k, ctypes.addressof(a), n) for k, a, n in ex._compiled], ex._ws_ptr, need)
        assert status == 0
    torch.cuda.synchronize()
    for _ in range(4):
        if short:
            assert d.lib.cdll.polar_b200_program_run(handle, torch.cuda.current_stream().cuda_stream) == 0
        else:
            ex.run()
        for row in rows:
            d.fmuon(*([eager[n][i] for n in row] for i in range(3)), lr=0.5, momentum=0.9, weight_decay=0.01, scale=0.7)
    torch.cuda.synchronize()
    assert d.device_status() == 0
    for n, (w, _, m) in eager.items():
        assert torch.equal(ex.t[n], w) and torch.equal(ex.t["m" + n], m)
    if short:
        d.lib.cdll.polar_b200_program_destroy(handle)
