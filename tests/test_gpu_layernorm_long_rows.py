"""flayernorm and flayernorm_grad on rows beyond 65536 columns: several stretches of rows, and sums whose rounding does not grow with the
row.

A thread adds 32 terms at a time in fp32 (U = 2^-24 for each of 32 additions at most), and such sums in 64 bits; the threads' sums are rounded to
fp32 and added in a tree of at most 16 steps: a sum is off by at most 32 + 1 + 16 < 50 times U of the sum of its terms' magnitudes, whatever the row's
length."""
import numpy as np
import pytest

from test_gpu_layernorm import EPS, U, close, env, expect_grad, inputs  # noqa: F401
from test_gpu_layernorm_means import expect_near

pytestmark = pytest.mark.gpu


def chain(cols):
    return 50


def grad_of(torch, x, g, gamma, mean, rstd):
    """As expect_grad, the row's sums with the chain of above."""
    want, off = expect_grad(torch, x, g, gamma, mean, rstd)
    x64, g64, m, r = x.double(), g.double(), mean.double()[:, None], rstd.double()[:, None]
    h, q = (x64 - m) * r, g64 * gamma.double()
    a, b = q.mean(1, keepdim=True), (q * h).mean(1, keepdim=True)
    off_a, off_b = (chain(0) + 3) * U * q.abs().mean(1, keepdim=True), (chain(0) + 7) * U * (q * h).abs().mean(1, keepdim=True)
    off_dx = r * (U * q.abs() + off_a + off_b * h.abs() + 3 * U * (h * b).abs() + 4 * U * (q.abs() + a.abs() + (h * b).abs())) + 2 * U * want[0].abs()
    return want, (off_dx, off[1], off[2])


@pytest.mark.parametrize("rows,cols", [(130, 65537), (70, 70001), (65, 65540), (9, 262144), (300, 66001), (1, 1 << 20)])
def test_against_the_formulas(env, rows, cols):  # noqa: F811
    torch, d = env
    x, g, gamma, beta = inputs(torch, rows, cols)
    nan = lambda *s: torch.full(s, np.nan, device="cuda")  # noqa: E731
    out, mean, rstd = nan(rows, cols), nan(rows), nan(rows)
    d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
    for got, want, off in zip((out, mean, rstd), *expect_near(torch, x, gamma, beta, chain=chain)):
        close(got, want, off)
    need = d.lib.cdll.polar_b200_flayernorm_grad_workspace_bytes(rows, cols)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    dx, dgamma, dbeta = nan(rows, cols), nan(cols), nan(cols)

    def call(din, bytes_):
        return d.lib.cdll.polar_b200_flayernorm_grad(g.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), rows, cols,
                                                     din.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), ws.data_ptr(), bytes_,
                                                     torch.cuda.current_stream().cuda_stream)

    assert call(dx, need) == 0 and call(dx, need - 1) == 5
    for got, want, off in zip((dx, dgamma, dbeta), *grad_of(torch, x, g, gamma, mean, rstd)):
        close(got, want, off)
    assert (ws[need:] == 255).all()
    sums = dgamma.clone(), dbeta.clone()
    dgamma.fill_(np.nan), dbeta.fill_(np.nan)
    assert call(x if rows % 2 else g, need) == 0             # in place: the same bits
    assert torch.equal(x if rows % 2 else g, dx) and torch.equal(dgamma, sums[0]) and torch.equal(dbeta, sums[1])


@pytest.mark.parametrize("cols", [1 << 20, (1 << 22) + 3, 1 << 25])
def test_long_sums_keep_their_digits(env, cols):  # noqa: F811
    # deviations of one size, whose squares a sum in fp32 would round alike again and again
    torch, d = env
    x = torch.full((1, cols), 0.55, device="cuda")
    x[0, ::2] = -0.55
    one, zero = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    out, mean, rstd = torch.empty_like(x), torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    d.flayernorm(x, one, zero, EPS, out, mean, rstd)
    for got, want, off in zip((out, mean, rstd), *expect_near(torch, x, one, zero, chain=chain)):
        close(got, want, off)
    # a gradient that is the same everywhere, on top of what follows the row
    g = torch.full_like(x, 0.3)
    g[0, ::2] = 0.9
    dx = torch.empty_like(x)
    d.flayernorm_grad(g, x, None, mean, rstd, dx)
    (want, _, _), (off, _, _) = grad_of(torch, x, g, one, mean, rstd)
    close(dx, want, off)
