"""flogprob of rows that are nearly certain of one class: the logarithm of its probability and the entropy are small numbers, and keep their digits.

U = 2^-24.  With d = x - max and s the sum of exp(d) over all but the largest element, the largest's log probability is -log1p(s) and the
entropy log1p(s) - t / (1 + s), t the sum of exp(d) d.  An exponential is off by U |d| from d's rounding, by U |d| from the product that makes it a power of two and by
4 U of its own, relative to itself; a sum by its chain of additions, classes / 32 + 40 at most; the logarithm, the quotient, product and difference by a
few U each.  Nothing is off by U of 1.  Exponentials below 2^-126 count as zero."""
import numpy as np
import pytest

from test_gpu_logprob import U, env, run  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(torch, rows, classes, ties=False):
    gen = torch.Generator(device="cuda").manual_seed(rows * 31 + classes)
    x = torch.randn((rows, classes), device="cuda", generator=gen)
    at = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
    r = torch.arange(rows, device="cuda")
    x[r, at] = x.amax(1) + torch.linspace(2, 60, rows, device="cuda")
    if ties:                                                 # a second one of the same
        other = (at + 1) % classes
        x[r, other] = x[r, at]
        at = torch.minimum(at, other)
    return x, at


def expect(torch, x, at):
    """Of the largest, at `at`: log probability, entropy, and how far they may be off."""
    d = x.double() - x.double().amax(1, keepdim=True)
    e = d.exp()
    e[torch.arange(len(at), device="cuda"), at] = 0
    s, t = e.sum(1), (e * d).sum(1)
    c = (x.shape[1] / 32 + 40) * U
    none = x.shape[1] * 2.0 ** -126
    off_s = c * s + (e * (2 * d.abs() + 5)).sum(1) * U + none
    off_t = c * t.abs() + (e * d.abs() * (2 * d.abs() + 7)).sum(1) * U + 90 * none
    log_sum = torch.log1p(s)
    off_log = off_s / (1 + s) + 4 * U * log_sum
    q = t / (1 + s)
    ent = log_sum - q
    return {"logprob": (-log_sum, off_log), "entropy": (ent, off_log + off_t / (1 + s) + q.abs() * (off_s + 3 * U) + 2 * U * ent)}


def close(got, want, off):
    worst = ((got.double() - want).abs() - 1.000001 * off).max().item()
    assert worst <= 0, (worst, ((got.double() - want).abs() / want.abs().clamp(min=1e-300)).max().item())


SHAPES = [(7, 2, 0), (65, 3, 3), (40, 10, 0), (33, 16, 5), (20, 17, 0), (20, 40, 20), (1000, 100, 0), (1000, 100, 5), (1000, 250, 0), (1000, 250, 32), (50, 500, 0),
          (1000, 400, 20), (300, 1000, 0), (300, 1000, 3), (2400, 3001, 0), (2400, 3001, 20), (2400, 8192, 5), (3, 9001, 0), (25, 9001, 5), (400, 9001, 20), (700, 9001, 0),
          (140, 15000, 5), (70, 30001, 0), (2, 131072, 0), (2, 131072, 20)]


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("rows,classes,top", SHAPES)
def test_small_logarithms_keep_their_digits(env, rows, classes, top, ties):  # noqa: F811
    torch, d = env
    x, at = rows_of(torch, rows, classes, ties)
    o = run(torch, d, x, at, top)
    want = expect(torch, x, at)
    close(o["logprob"], *want["logprob"])
    close(o["entropy"], *want["entropy"])
    if top:
        assert torch.equal(o["top_ids"][:, 0], at)
        close(o["top_logprob"][:, 0], *want["logprob"])


@pytest.mark.parametrize("classes", [2, 16, 100, 250, 1000, 3001, 9001])
def test_one_class_left(env, classes):  # noqa: F811
    # all others shut out, by -inf or by the type's lowest value: certain, to the bit
    torch, d = env
    for shut in (-np.inf, float(np.finfo(np.float32).min)):
        x = torch.full((5, classes), shut, device="cuda")
        at = torch.tensor([0, 1, classes - 1, classes // 2, 1], device="cuda")
        x[torch.arange(5, device="cuda"), at] = torch.tensor([0.0, -3.0, 80.0, 1e-3, 5.0], device="cuda")
        o = run(torch, d, x, at, 0)
        assert not o["logprob"].any() and not o["entropy"].any()
        assert o["logsumexp"].tolist() == x[torch.arange(5, device="cuda"), at].tolist()
