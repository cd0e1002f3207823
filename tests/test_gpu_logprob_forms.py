"""flogprob against its formulas at sizes that between them reach the kernels that the sizes of test_gpu_logprob.py do not: CTAs of 128 and 256
threads per row, clusters of two and four CTAs, a warp's row of four chunks and more, parts of a warp without alternatives; with ties, masks and NaN
among many such rows, and rows whose offset passes 32 bits."""
import numpy as np
import pytest

from test_gpu_logprob import U, close, edge_rows, env, expect, expect_grad, logits, run  # noqa: F401

pytestmark = pytest.mark.gpu


def best(torch, x, top):
    """The `top` largest of each row, ties to the lowest index, NaN above all."""
    return torch.sort(x + 0.0, dim=1, descending=True, stable=True)[1][:, :top]


def check(torch, x, ids, o, top):
    for i in range(0, x.shape[0], 256):                      # (a few rows at a time: they are held in 64 bits several times over)
        part = slice(i, i + 256)
        want = expect(torch, x[part], ids[part])
        for k in ("logprob", "entropy", "logsumexp"):
            close(o[k][part], *want[k])
        if top:
            at = best(torch, x[part], top)
            assert torch.equal(o["top_ids"][part].long(), at)
            d, log_sum, off_log = want["parts"]
            dt = torch.gather(d, 1, at)
            w = dt - log_sum[:, None]
            close(o["top_logprob"][part], w, U * dt.abs() + off_log[:, None] + U * w.abs())


def test_the_order_of_the_expected_alternatives(env):  # noqa: F811
    torch, _ = env
    x = torch.tensor([[0.0, -0.0, 2.0, np.nan, 2.0, -np.inf, np.nan, np.inf]], device="cuda")
    assert best(torch, x, 8).tolist() == [[3, 6, 7, 2, 4, 0, 1, 5]]


@pytest.mark.parametrize("rows,classes,top", [
    (400, 9001, 5), (500, 12000, 32), (297, 1025, 20), (592, 29573, 0),               # 256 threads
    (700, 9001, 20), (700, 9001, 0), (593, 1030, 32), (900, 8193, 1), (600, 70000, 9),  # 128 threads
    (140, 15000, 5), (140, 15001, 0), (70, 30000, 32), (70, 30001, 0),                # two and four CTAs
    (2400, 3001, 20), (2400, 3001, 0), (2400, 8191, 5), (2368, 8192, 32), (2500, 4097, 1), (2400, 2049, 12),   # a warp, four chunks and more
    (1000, 100, 0), (1000, 200, 0), (889, 17, 0), (1000, 125, 8), (1000, 253, 0), (889, 126, 9)])              # 8 and 16 lanes
def test_forward(env, rows, classes, top):  # noqa: F811
    torch, d = env
    x, ids = logits(torch, rows, classes)
    check(torch, x, ids, run(torch, d, x, ids, top), top)


@pytest.mark.parametrize("rows,classes,pitch,offset,top", [(400, 9001, 9004, 1, 20), (700, 9001, 9003, 2, 5), (140, 15001, 15001, 3, 9), (2400, 3001, 3004, 1, 20),
                                                           (1000, 100, 101, 1, 0), (1000, 200, 203, 3, 20)])
def test_rows_apart_and_on_odd_boundaries(env, rows, classes, pitch, offset, top):  # noqa: F811
    torch, d = env
    x, ids = logits(torch, rows, classes, pitch=pitch, offset=offset)
    for kind in (torch.int32, torch.float32):
        check(torch, x, ids, run(torch, d, x, ids, top, kind), top)


@pytest.mark.parametrize("rows,classes", [(400, 9001), (700, 9001), (700, 1030), (140, 15000), (70, 30001), (2400, 3001), (2400, 8192), (2400, 2050)])
def test_edges_among_many_rows(env, rows, classes):  # noqa: F811
    torch, d = env
    for top, at in ((5, 0), (20, rows // 2), (32, rows - 14)):   # the edges in front, in the middle, at the end
        x, ids = logits(torch, rows, classes, offset=at % 4)
        edge_rows(x[at:], ids[at:], classes)
        shut, nan, inf = at + 2, rows // 3, rows // 3 + 1
        x[nan, classes - 1], x[inf, 7] = np.nan, np.inf
        x[rows // 3 + 2, 40:] = -np.inf                      # fewer left than some alternatives, all in front
        ids[rows // 3 + 2] = 11
        ids[rows // 3 + 3] = -1
        o = run(torch, d, x, ids, top)
        keep = torch.tensor([i for i in range(rows) if i not in (shut, nan, inf, rows // 3 + 3)], device="cuda")
        check(torch, x[keep], ids[keep], {k: v[keep] for k, v in o.items()}, top)
        assert o["logprob"][rows // 3 + 3] == 0 and o["logprob"][shut] == -np.inf and o["entropy"][shut] == 0 and o["logsumexp"][shut] == -np.inf
        assert o["top_ids"][shut].tolist() == list(range(top)) and (o["top_logprob"][shut] == -np.inf).all()
        for r in (nan, inf):
            assert torch.isnan(o["logprob"][r]) and torch.isnan(o["entropy"][r]) and torch.isnan(o["logsumexp"][r])
            assert torch.equal(o["top_ids"][r:r + 1], best(torch, x[r:r + 1], top))


@pytest.mark.parametrize("rows,classes,pitch", [(5, 40000, 1 << 30), (600, 9001, (1 << 23) + 1), (2400, 3001, (1 << 21) + 3)])
def test_rows_beyond_32_bits_of_offset(env, rows, classes, pitch):  # noqa: F811
    torch, d = env
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("not enough free memory")
    assert (rows - 1) * pitch + classes >= 1 << 32
    x, ids = logits(torch, rows, classes, pitch=pitch)
    o = run(torch, d, x, ids, 9)
    check(torch, x, ids, o, 9)
    g, ge = torch.ones(rows, device="cuda"), torch.full((rows,), 0.5, device="cuda")
    dx = torch.empty((rows, classes), device="cuda")
    d.flogprob_grad(x, ids, o["logsumexp"], o["entropy"], g, ge, dx)
    want, off = expect_grad(torch, x, ids, o["logsumexp"], o["entropy"], g, ge)
    close(dx, want, off)
    d.flogprob_grad(x, ids, o["logsumexp"], o["entropy"], g, ge, x)   # in place, across the pitch
    assert torch.equal(x, dx)
