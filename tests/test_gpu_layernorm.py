"""flayernorm and flayernorm_grad against their formulas in 64 bits.

Tolerances count roundings: U = 2^-24 is half a step of fp32 relative to the value.  A sum of n terms in which no chain of additions is longer
than c is off by at most c * U times the sum of the terms' magnitudes.  A row's sums have chains of at most cols / 32 + 16 additions (a
warp's lane, then a tree); a sum over rows of at most rows / 64 + 600 (a stretch of rows, then the stretches)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module")
def env():
    import torch
    import __graft_entry__ as ge
    ge.load_package()
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return torch, DeviceBuiltins()


def inputs(torch, rows, cols, seed=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(rows * 7919 + cols + seed)
    new = lambda *s: torch.randn(int(np.prod(s)) + offset, device="cuda", generator=g)[offset:].view(s)  # noqa: E731
    x = new(rows, cols)
    if rows:
        x.mul_(torch.rand((rows, 1), device="cuda", generator=g) + 0.5).add_(torch.randn((rows, 1), device="cuda", generator=g))
    return x, new(rows, cols), new(cols), new(cols)


def expect(torch, x, gamma, beta, eps=EPS):
    """The formula, and how far a result may be off."""
    x64 = x.double()
    mean = x64.mean(1)
    d = x64 - mean[:, None]
    var = (d * d).mean(1)
    rstd = 1 / (var + eps).sqrt()
    out = d * rstd[:, None] * gamma.double() + beta.double()
    c = (x.shape[1] / 32 + 16) * U
    off_mean = c * x64.abs().mean(1) + U * mean.abs()
    # a mean that is off by e moves each deviation by e and the variance by e^2 (its first order sums to nothing); a deviation is
    # rounded once; rstd has half the variance's relative error and the roundings of the square root and the quotient
    off_rstd = rstd * (0.5 * (c + 4 * U + off_mean ** 2 * rstd ** 2) + 4 * U)
    scale = (gamma.double().abs() * rstd[:, None])
    off = scale * (off_mean[:, None] + U * d.abs() + U * x64.abs()) + (off_rstd / rstd)[:, None] * (d * scale).abs() \
        + 4 * U * (d * scale).abs() + U * out.abs()
    return (out, mean, rstd), (off, off_mean, off_rstd)


def close(got, want, off):
    """Within the tolerance, which gets a millionth for its own rounding, and a least magnitude."""
    d = (got.double() - want).abs()
    worst = (d - 1.000001 * off - 1e-37).max().item() if d.numel() else 0.0
    assert worst <= 0, (worst, d.max().item())


SIZES = [(1, 1), (3, 1), (5, 2), (4, 3), (33, 7), (70, 13), (9, 32), (5, 33), (130, 64), (3, 100), (77, 128), (6, 129), (31, 255), (40, 256),
         (1000, 260), (999, 514), (300, 1000), (5, 1024), (257, 1511), (64, 2048), (2, 4093), (1, 4096), (500, 4096), (3, 5000),
         (17, 8192), (2, 9001), (3, 16384), (2, 16388), (2, 20001), (1, 32768), (2, 32772), (1, 70001),
         (2400, 2050), (2500, 3099), (2370, 4095), (600, 4101), (700, 6145), (900, 8191), (620, 8193), (610, 12289), (600, 16383),
         (200, 9001), (150, 24001), (90, 28010), (3, 45000), (2, 53001), (40, 60001),
         (2001, 1511), (400, 1033), (310, 2101), (320, 2701), (310, 3583), (300, 4301), (350, 6001), (310, 7001),
         (300, 16385), (310, 20481), (300, 24577), (297, 28671)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward(env, rows, cols):
    torch, d = env
    x, _, gamma, beta = inputs(torch, rows, cols)
    out, mean, rstd = torch.full_like(x, np.nan), torch.full((rows,), np.nan, device="cuda"), torch.full((rows,), np.nan, device="cuda")
    d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
    for g, w, o in zip((out, mean, rstd), *expect(torch, x, gamma, beta)):
        close(g, w, o)
    # without what may be left out: the same bits
    bare, ones, zeros = torch.empty_like(x), torch.ones_like(gamma), torch.zeros_like(beta)
    d.flayernorm(x, None, None, EPS, bare)
    d.flayernorm(x, ones, zeros, EPS, out)
    assert torch.equal(bare, out)
    d.flayernorm(x, ones, zeros, EPS, x)                     # in place
    assert torch.equal(x, out)


def expect_grad(torch, x, g, gamma, mean, rstd):
    x64, g64, m, r = x.double(), g.double(), mean.double()[:, None], rstd.double()[:, None]
    h, q = (x64 - m) * r, g64 * gamma.double()
    a, b = q.mean(1, keepdim=True), (q * h).mean(1, keepdim=True)
    dx = r * (q - a - h * b)
    c = (x.shape[1] / 32 + 16) * U
    # h: a rounded difference and product; the rest as its terms come
    off_h = 3 * U * h.abs()
    off_a, off_b = (c + 3 * U) * q.abs().mean(1, keepdim=True), (c + 7 * U) * (q * h).abs().mean(1, keepdim=True)
    off_dx = r * (U * q.abs() + off_a + off_b * h.abs() + off_h * b.abs() + 4 * U * (q.abs() + a.abs() + (h * b).abs())) + 2 * U * dx.abs()
    cr = (x.shape[0] / 64 + 600) * U
    return (dx, (g64 * h).sum(0), g64.sum(0)), (off_dx, (cr + 5 * U) * (g64 * h).abs().sum(0), cr * g64.abs().sum(0))


@pytest.mark.parametrize("rows,cols", SIZES)
def test_backward(env, rows, cols):
    torch, d = env
    x, g, gamma, beta = inputs(torch, rows, cols)
    mean, rstd = x.mean(1), 1 / (x.var(1, unbiased=False) + EPS).sqrt()
    nan = lambda *s: torch.full(s, np.nan, device="cuda")  # noqa: E731
    dx, dgamma, dbeta = nan(rows, cols), nan(cols), nan(cols)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx, dgamma, dbeta)
    for got, want, off in zip((dx, dgamma, dbeta), *expect_grad(torch, x, g, gamma, mean, rstd)):
        close(got, want, off)
    # parts of it, twice, and in place: the same bits
    dx2, dg2, db2 = nan(rows, cols), nan(cols), nan(cols)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx2)
    assert torch.equal(dx, dx2)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx2, None, db2)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx2, dg2)
    assert torch.equal(dx, dx2) and torch.equal(dgamma, dg2) and torch.equal(dbeta, db2)
    for into in (0, 1):
        pair = [g.clone(), x.clone()]
        dg2, db2 = nan(cols), nan(cols)
        d.flayernorm_grad(*pair, gamma, mean, rstd, pair[into], dg2, db2)
        assert torch.equal(pair[into], dx) and torch.equal(dgamma, dg2) and torch.equal(dbeta, db2)
    d.flayernorm_grad(g, x, None, mean, rstd, dx2)
    d.flayernorm_grad(g, x, torch.ones_like(gamma), mean, rstd, dx)
    assert torch.equal(dx, dx2)


@pytest.mark.parametrize("rows,cols", [(5, 36), (3, 512), (7, 4096), (2, 20000), (2400, 4096), (600, 8192), (600, 9000)])
def test_tensors_on_odd_boundaries(env, rows, cols):
    torch, d = env
    for offset in (1, 2, 3):
        x, g, gamma, beta = inputs(torch, rows, cols, offset=offset)
        assert x.data_ptr() % 16
        out = torch.empty(rows * cols + offset, device="cuda")[offset:].view(rows, cols)
        mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
        for got, want, off in zip((out, mean, rstd), *expect(torch, x, gamma, beta)):
            close(got, want, off)
        dgamma, dbeta = torch.empty(cols + offset, device="cuda")[offset:], torch.empty(cols + offset, device="cuda")[offset:]
        d.flayernorm_grad(g, x, gamma, mean, rstd, out, dgamma, dbeta)
        for got, want, off in zip((out, dgamma, dbeta), *expect_grad(torch, x, g, gamma, mean, rstd)):
            close(got, want, off)


def test_gradient_against_differences(env):
    # of a fixed weighting of the outputs, in 64 bits on the host, at every input and weight
    torch, d = env
    x, g, gamma, beta = inputs(torch, 6, 37)
    out, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx, dgamma, dbeta)
    leaves = [t.double().cpu() for t in (x, gamma, beta)]

    def value():
        lx, lg, lb = leaves
        dev = lx - lx.mean(1, keepdim=True)
        return ((dev / (dev.square().mean(1, keepdim=True) + EPS).sqrt() * lg + lb) * g.double().cpu()).sum().item()

    for leaf, grad in zip(leaves, (dx, dgamma, dbeta)):
        flat = leaf.view(-1)
        for i in range(flat.numel()):
            at = flat[i].item()
            flat[i] = at + 1e-5
            up = value()
            flat[i] = at - 1e-5
            down = value()
            flat[i] = at
            # differences: third derivatives times 1e-10, and 2^-53 of the sum over 2e-5; the kernel: some 30 roundings of terms below 100
            assert abs((up - down) / 2e-5 - grad.reshape(-1)[i].item()) < 2e-4


def test_rows_and_values_at_the_edges(env):
    torch, d = env
    # no rows: sums of nothing
    dgamma, dbeta = torch.ones(40, device="cuda"), torch.ones(40, device="cuda")
    empty, none = torch.empty((0, 40), device="cuda"), torch.empty(0, device="cuda")
    d.flayernorm(empty, torch.ones(40, device="cuda"), None, EPS, empty)
    d.flayernorm_grad(empty, empty, None, none, none, empty, dgamma, dbeta)
    assert not dgamma.any() and not dbeta.any()
    # a constant row has variance 0; NaN and infinities stay in their rows
    for cols in (48, 300, 5000, 40000):
        x = torch.randn((6, cols), device="cuda")
        x[1] = 3.0
        x[2, 5], x[3, cols - 1], x[4, 0] = np.nan, np.inf, -np.inf
        out, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
        d.flayernorm(x, None, None, EPS, out, mean, rstd)
        assert torch.equal(out[1], torch.zeros_like(out[1])) and mean[1] == 3.0
        assert torch.isnan(out[2:5]).all() and torch.isfinite(out[[0, 1, 5]]).all()
    # a row far from zero: the deviations are taken around the mean
    x = torch.randn((4, 1024), device="cuda") + 4096.0
    out, one, zero = torch.empty_like(x), torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
    d.flayernorm(x, one, zero, EPS, out)
    (want, _, _), (off, _, _) = expect(torch, x, one, zero)
    close(out, want, off)


def test_sums_over_many_rows_on_a_given_workspace(env):
    torch, d = env
    for rows, cols in ((20000, 24), (3000, 512), (40, 20000)):
        x, g, gamma, _ = inputs(torch, rows, cols)
        mean, rstd = x.mean(1), 1 / (x.var(1, unbiased=False) + EPS).sqrt()
        dx, dgamma, dbeta = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
        need = d.lib.cdll.polar_b200_flayernorm_grad_workspace_bytes(rows, cols)
        ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.current_stream().cuda_stream
        call = lambda bytes_: d.lib.cdll.polar_b200_flayernorm_grad(  # noqa: E731
            g.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), rows, cols, dx.data_ptr(), dgamma.data_ptr(),
            dbeta.data_ptr(), ws.data_ptr(), bytes_, stream)
        assert call(need) == 0
        for got, want, off in zip((dx, dgamma, dbeta), *expect_grad(torch, x, g, gamma, mean, rstd)):
            close(got, want, off)
        assert (ws[need:] == 255).all()
        assert call(need - 1) == 5


def test_two_streams_and_a_captured_call(env):
    torch, d = env
    x, g, gamma, beta = inputs(torch, 300, 1024)
    mean, rstd = x.mean(1), 1 / (x.var(1, unbiased=False) + EPS).sqrt()
    want = [torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)]
    d.flayernorm_grad(g, x, gamma, mean, rstd, *want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(t) for t in want] for _ in streams]
    for _ in range(20):
        for s, o in zip(streams, got):
            with torch.cuda.stream(s):
                d.flayernorm_grad(g, x, gamma, mean, rstd, *o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))
    graphs, outs = [], []
    for _ in range(2):                                       # two graphs, each with scratch of its own
        outs.append([torch.zeros_like(t) for t in want])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            d.flayernorm_grad(g, x, gamma, mean, rstd, *outs[-1])
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("rows,cols", [(700, 9001), (300, 20000), (2400, 2050)])
def test_long_rows_captured_and_on_two_streams(env, rows, cols):
    torch, d = env
    x, g, gamma, beta = inputs(torch, rows, cols)

    def call(o):
        d.flayernorm(x, gamma, beta, EPS, *o[:3])
        d.flayernorm_grad(g, x, gamma, o[1], o[2], *o[3:])

    new = lambda: [torch.zeros_like(t) for t in (x, x[:, 0].contiguous(), x[:, 0].contiguous(), x, gamma, beta)]  # noqa: E731
    captured, got = new(), [new(), new()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                            # (before any other call of this shape)
        call(captured)
    torch.cuda.synchronize()
    for o in got:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(3):
                call(o)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, captured))
