"""flayernorm and flayernorm_grad against their formulas in 64 bits at sizes that between them reach every form of their kernels that the
sizes of test_gpu_layernorm.py do not: full batches of vectors and of rows off 16-byte boundaries, clusters of every size."""
import numpy as np
import pytest

from test_gpu_layernorm import EPS, close, env, expect, expect_grad, inputs  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, columns, whether the rows are on 16-byte boundaries
FORWARD_SHAPES = [
    (172, 24684, True), (1, 404, True), (3861, 1087, False), (3945, 1064, True), (2448, 1715, False), (2055, 2044, True), (1027, 4096, True),
    (297, 95, False), (297, 108, True), (24675, 170, False), (26217, 160, True), (16983, 247, False), (16387, 256, True), (1, 527, False),
    (297, 1424, True), (1523, 2759, False), (2369, 2272, True), (1363, 3082, False), (1173, 3584, True), (735, 5728, True), (598, 7044, True),
    (1, 79, False), (297, 204, False), (297, 144, True), (11952, 351, False), (14172, 296, True), (9779, 429, False), (10702, 392, True),
    (8068, 520, True), (6171, 680, True), (4996, 840, True), (525, 8030, False), (297, 264, False), (6639, 632, False), (4404, 953, False),
    (297, 48, False), (297, 52, True), (53095, 79, False), (43693, 96, True), (34666, 121, False), (41946, 100, True)]
BACKWARD_SHAPES = [(1, 11960, True), (30, 22856, True), (50, 24756, True), (40, 32082, False), (20, 34407, False), (30, 44006, False), (20, 54012, True),
                   (25, 59328, True), (3000, 86, False), (200, 12000, True), (64, 28004, True), (33, 65536, True), (20, 65535, False)]


def tensors(torch, rows, cols, aligned):
    x, g, gamma, beta = inputs(torch, rows, cols, offset=0 if aligned else 1)
    assert not aligned or (cols % 4 == 0 and x.data_ptr() % 16 == 0)
    assert aligned or cols % 4 or x.data_ptr() % 16
    return x, g, gamma, beta


@pytest.mark.parametrize("rows,cols,aligned", FORWARD_SHAPES)
def test_forward(env, rows, cols, aligned):  # noqa: F811
    torch, d = env
    x, _, gamma, beta = tensors(torch, rows, cols, aligned)
    out, mean, rstd = torch.full_like(x, np.nan), torch.full((rows,), np.nan, device="cuda"), torch.full((rows,), np.nan, device="cuda")
    d.flayernorm(x, gamma, beta, EPS, out, mean, rstd)
    for got, want, off in zip((out, mean, rstd), *expect(torch, x, gamma, beta)):
        close(got, want, off)
    bare = torch.empty_like(x)
    d.flayernorm(x, None, None, EPS, bare)
    d.flayernorm(x, torch.ones_like(gamma), torch.zeros_like(beta), EPS, x)   # in place
    assert torch.equal(bare, x)


@pytest.mark.parametrize("rows,cols,aligned", BACKWARD_SHAPES)
def test_backward(env, rows, cols, aligned):  # noqa: F811
    torch, d = env
    x, g, gamma, beta = tensors(torch, rows, cols, aligned)
    mean, rstd = x.mean(1), 1 / (x.var(1, unbiased=False) + EPS).sqrt()
    nan = lambda *s: torch.full(s, np.nan, device="cuda")  # noqa: E731
    dx, dgamma, dbeta = nan(rows, cols), nan(cols), nan(cols)
    d.flayernorm_grad(g, x, gamma, mean, rstd, dx, dgamma, dbeta)
    for got, want, off in zip((dx, dgamma, dbeta), *expect_grad(torch, x, g, gamma, mean, rstd)):
        close(got, want, off)
    for into in (0, 1):                                      # in place: the same bits
        pair = [g.clone(), x.clone()] if aligned else [g, x]
        if not aligned and into:
            continue
        dg2, db2 = nan(cols), nan(cols)
        d.flayernorm_grad(*pair, gamma, mean, rstd, pair[into], dg2, db2)
        assert torch.equal(pair[into], dx) and torch.equal(dgamma, dg2) and torch.equal(dbeta, db2)
