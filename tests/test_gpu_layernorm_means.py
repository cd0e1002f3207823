"""flayernorm's means: rows that are constant or far from zero, in every kind of kernel.

U = 2^-24 is half a step of fp32.  With m a first mean of the row, d = x - m is rounded once (U |d|; not at all where the row is
constant, since m lies within a factor of two of it), and the mean of d corrects both m and the sum of squares.  So no error of the size of
|x| reaches a deviation: c, the mean of d, is off by its sum's chain of additions (`chain`, at most cols / 32 + 16 of them) and the quotient's rounding,
relative to the mean of |d|."""
import numpy as np
import pytest

from test_gpu_layernorm import EPS, U, close, env  # noqa: F401

pytestmark = pytest.mark.gpu


def chain_of(cols):
    return cols / 32 + 16


def expect_near(torch, x, gamma, beta, eps=EPS, chain=chain_of):
    """The formula, and how far out, mean and rstd may be off."""
    x64 = x.double()
    mean = x64.mean(1)
    d = x64 - mean[:, None]
    var = (d * d).mean(1)
    rstd = 1 / (var + eps).sqrt()
    g = gamma.double()
    out = d * rstd[:, None] * g + beta.double()
    k = chain(x.shape[1])
    c = (k + 2) * U * x64.abs().mean(1)                      # how far the first mean may be off
    size = d.abs().mean(1) + c                               # the mean of |x - m| at most
    off_d = ((k + 3) * U * size)[:, None] + U * (2 * d.abs() + 2 * c[:, None])
    # the squares' sum is around m: what is taken off again is c^2
    off_var = (k + 6) * U * (var + c * c) + 2 * c * (k + 3) * U * size + 2 * U * c * c
    off_rstd = rstd * (0.5000001 * off_var / (var + eps) + 4 * U)
    scale = g.abs() * rstd[:, None]
    off = scale * off_d + (off_rstd / rstd)[:, None] * (d * scale).abs() + 4 * U * ((d * scale).abs() + scale * off_d) + U * out.abs()
    return (out, mean, rstd), (off, (k + 3) * U * size + U * c + U * mean.abs(), off_rstd)


# one of each kind: lanes of a warp, a warp, a CTA, a cluster; the ring of rows off 16-byte boundaries; beyond 65536 columns
SHAPES = [(3, 7), (9, 41), (40, 128), (600, 300), (5, 1000), (4200, 1000), (33, 1511), (2400, 2101), (2, 4100), (1100, 4096), (7, 7680), (600, 7830), (2, 9001),
          (600, 9001), (300, 20001), (3, 16384), (2, 20000), (200, 32000), (1, 30000), (2, 45001), (3, 48000), (2, 70001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_constant_rows(env, rows, cols):  # noqa: F811
    # all deviations are the same whole number of steps, so their sum and its quotient by cols are exact: nothing is left of them
    torch, d = env
    values = torch.tensor([3.0, 1000.0, 1000.3, -0.1, 777.77, 0.0, 1e-3], device="cuda")[torch.arange(rows, device="cuda") % 7]
    x = values[:, None].expand(rows, cols).contiguous()
    gen = torch.Generator(device="cuda").manual_seed(cols)
    gamma, beta = torch.randn(cols, device="cuda", generator=gen), torch.randn(cols, device="cuda", generator=gen)
    out, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
    assert torch.equal(mean, values)
    assert torch.equal(out, beta.expand(rows, cols))
    (_, _, want), (_, _, off) = expect_near(torch, x, gamma, beta)
    close(rstd, want, off)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rows_far_from_zero(env, rows, cols):  # noqa: F811
    torch, d = env
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    new = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    at = torch.tensor([1000.3, -4097.7, 33.3, 0.0], device="cuda")[torch.arange(rows, device="cuda") % 4]
    x, gamma, beta = new(rows, cols) * 0.05 + at[:, None], new(cols), new(cols)
    out, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
    for got, want, off in zip((out, mean, rstd), *expect_near(torch, x, gamma, beta)):
        close(got, want, off)


def test_values_that_are_none_and_no_eps(env):  # noqa: F811
    # NaN and infinities as before, and no variance below zero where a row is all but constant
    torch, d = env
    for cols in (41, 1000, 9001, 45001):
        x = torch.full((6, cols), 1000.3, device="cuda")
        x[0, cols // 2], x[1, 1], x[2, 0] = np.nan, np.inf, -np.inf
        x[4] = torch.randn(cols, device="cuda")
        out, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
        d.flayernorm(x, None, None, 1e-30, out, mean, rstd)
        assert torch.isnan(out[:3]).all() and torch.isnan(rstd[:3]).all()
        assert not out[[3, 5]].any() and torch.isfinite(rstd[3:]).all() and (rstd[3:] > 0).all()


def test_deviations_whose_squares_are_beyond_fp32(env):  # noqa: F811
    # of a constant row the first mean may be a step off, whose square is infinite here: still nothing is left of it
    torch, d = env
    for cols in (7, 41, 1000, 9001, 20001, 45001, 70001):
        x = torch.tensor([1e30, -1.1e30, 7.7e29], device="cuda")[:, None].repeat(1, cols)
        beta = torch.randn(cols, device="cuda")
        out, mean, rstd = torch.empty_like(x), torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
        d.flayernorm(x, None, beta, EPS, out, mean, rstd)
        assert torch.equal(out, beta.expand(3, cols)) and torch.equal(mean, x[:, 0].contiguous()) and (rstd >= 0).all()
