"""The loss of pairs where a pair's rewards lie far or infinitely far apart: a chosen or rejected token whose logit was masked has a log probability
of minus infinity, and where the smoothing leaves one side of the loss, that side is as exact as it is small."""
import math

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from test_gpu_sequence_losses import U, batch, up  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def run(d, b, **k):
    loss, r, g = (torch.full((n,), math.nan, device="cuda:0") for n in (3, len(b["offsets"]) - 1, len(b["ids"])))
    d.fpreference_loss(up(b["logprob"]), up(b["ids"]), up(b["offsets"]), loss, r, g, **k)
    return loss.cpu().numpy().astype(np.float64), r.cpu().numpy(), g.cpu().numpy()


def terms(z, smoothing):
    """The two sides of the loss; one of weight zero is none, whatever it is."""
    sides = ((1 - smoothing, np.logaddexp(0, -z)), (smoothing, np.logaddexp(0, z)))
    return sum(np.where(by > 0, by * side, 0.0) if by > 0 else np.zeros(len(z)) for by, side in sides)


# one CTA, few and many sequences to it; three kernels, with a warp and with a lane for each sequence
@pytest.mark.parametrize("tokens,pairs", [(40, 3), (3000, 200), (30000, 8), (20000, 3000)])
@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("average", [False, True])
def test_a_token_of_probability_zero(d, tokens, pairs, smoothing, side, average):
    b = batch(50 + pairs, tokens, 2 * pairs, counted=0.9, empty_rows=False)
    b["offsets"] = np.linspace(0, tokens, 2 * pairs + 1).astype(np.int64)
    b["ids"][b["offsets"][:-1]] = 5                          # each sequence has a token that counts
    at = int(b["offsets"][2 + side])                         # in the second pair
    b["logprob"][at] = -np.inf
    loss, r, g = run(d, b, smoothing=smoothing, average=average, beta=0.5)
    of = np.repeat(np.arange(2 * pairs), np.diff(b["offsets"]))
    counts = b["ids"] >= 0
    n = np.bincount(of[counts], minlength=2 * pairs)
    assert n.min() > 0
    sums = np.array([b["logprob"][(of == s) & counts].astype(np.float64).sum() for s in range(2 * pairs)]) / (n if average else 1)
    z = 0.5 * (sums[0::2] - sums[1::2])
    assert z[1] == (-np.inf if side == 0 else np.inf) and np.isfinite(np.delete(z, 1)).all()
    each = terms(z, smoothing)
    expected = each.sum() / pairs
    infinite = (smoothing < 1) if side == 0 else (smoothing > 0)
    assert np.isinf(expected) == infinite
    # (as in the test of finite gaps: z's rounding and some eight operations to a pair, then some twenty additions)
    assert loss[0] == np.inf if infinite else abs(loss[0] - expected) <= 32 * U * np.delete(each + np.abs(z), 1).sum() / pairs
    assert loss[2] == z[1] and abs(loss[1] - (z > 0).mean()) <= 4 * U
    assert r[2 + side] == -np.inf and np.isfinite(np.delete(r, 2 + side)).all()
    # the gradient is one side's whole weight: the sigmoids are 0 and 1
    slope = -(1 - smoothing) if side == 0 else smoothing
    share = np.array([slope, -slope]) * 0.5 / pairs / (n[2:4] if average else 1)
    for s in (0, 1):
        its = g[(of == 2 + s) & counts]
        assert (np.abs(its - share[s]) <= 8 * U * abs(share[s])).all()
    assert np.isfinite(g).all() and (g[~counts] == 0).all()


@pytest.mark.parametrize("pairs", [1, 40, 3000])
@pytest.mark.parametrize("z", [-30.0, -20.0, -10.0, -1.0, 0.0, 1.0, 10.0, 20.0, 30.0])
@pytest.mark.parametrize("smoothing", [0.0, 0.5, 1.0])
def test_the_small_side_of_the_loss_keeps_its_digits(d, pairs, z, smoothing):
    lp = np.tile(np.array([z / 2, -z / 2], np.float32) - 20, pairs)
    b = {"logprob": lp, "ids": np.ones(2 * pairs, np.int64), "offsets": np.arange(2 * pairs + 1)}
    loss, _, g = run(d, b, smoothing=smoothing, beta=1.0)
    expected = terms(np.array([z]), smoothing)[0]
    # log1p and the exponential (4 steps and the argument's none: z is exact), four products and sums of what is not below zero; some twenty additions, a division
    assert abs(loss[0] - expected) <= 32 * U * expected
    slope = smoothing / (1 + math.exp(-z)) - (1 - smoothing) / (1 + math.exp(z))
    size = max(smoothing / (1 + math.exp(-z)), (1 - smoothing) / (1 + math.exp(z)))
    assert (np.abs(g * pairs - np.tile([slope, -slope], pairs)) <= 16 * U * size).all()
