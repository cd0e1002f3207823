"""How many digits orthogonalised momentum keeps.  Of a diagonal matrix every entry is a singular value by itself, and every sum of a product has one term,
so that each entry can be held to the bound of its own roundings, in units u = 2^-24:

  a pair      hi has 11 bits and lo the next 11: off by up to 2^-22, 4 u
  a product   its operands' errors, lo lo that is left out (4 u), three additions that are cut (2 u each) and one rounding: 11 u
  X           the quotient's rounding, 1 u, and a pair's
  G = X X     2 e(X) + 11 + 4,  as a pair
  P           a + b G + c G G: |b| G (e(G) + 2) + c G^2 (2 e(G) + 11 + 2) + 2 (|a| + |b| G + c G^2), over |P|, and a pair's 4
  P X         e(P) + 11, and 4 as a pair or 3 as it is taken off the weights; and e(X) as it passes the whole round, |s p'(s) / p(s)| e(X), for which
              e(P) counts only what G has beyond 2 e(X)."""
import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from test_gpu_muon import CLOSE, check, make, step  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
A, B, C = (float(np.float32(v)) for v in (3.4445, -4.7750, 2.0315))


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def rounds(s, steps):
    """The singular values after the rounds, and what they may be off by in u."""
    e = np.full(len(s), 5.0)
    for i in range(steps):
        g = s * s
        terms, p = A + abs(B) * g + C * g * g, A + B * g + C * g * g
        own = 15.0                                           # of G, beyond what X has
        of_p = (abs(B) * g * (own + 2) + C * g * g * (2 * own + 13) + 2 * terms) / abs(p) + 4
        e = e * np.abs(1 + 2 * g * (B + 2 * C * g) / p) + of_p + 11 + (4 if i + 1 < steps else 3)
        s = s * p
    return s, e


# one CTA's matrices, products, narrow matrices; beyond one round only those whose rounds are taken one by one
@pytest.mark.parametrize("shape,steps", [((64, 64), 1), ((100, 128), 1), ((128, 200), 1), ((200, 90), 1), ((200, 200), 1), ((300, 260), 1), ((64, 2000), 1), ((1500, 100), 1),
                                         ((400, 1000), 1), ((1000, 400), 1), ((1024, 1024), 1), ((64, 64), 2), ((100, 128), 5), ((200, 200), 2), ((300, 260), 5), ((900, 700), 3)])
def test_each_singular_value_by_itself(d, shape, steps):
    n = min(shape)
    rng = np.random.default_rng(sum(shape) + steps)
    v = (10.0 ** rng.uniform(-2, 0, n) * rng.choice([-1.0, 1.0], n)).astype(np.float32)
    g = torch.zeros(shape, device="cuda")
    at = torch.arange(n, device="cuda")
    g[at, at] = torch.from_numpy(v).cuda()
    w, m = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    d.fmuon([w], [g], [m], lr=1.0, momentum=0.0, nesterov=False, steps=steps, scale=1.0)
    torch.cuda.synchronize()
    assert d.device_status() == 0 and torch.equal(m, g)
    s = v.astype(np.float64) / np.sqrt((v.astype(np.float64) ** 2).sum())
    want, e = rounds(s, steps)
    got = -w[at, at].double().cpu().numpy()
    # (a lo of s below 2^-18 would lie among fp16's subnormal numbers; these are above)
    assert np.abs(s).min() > 2.0 ** -18
    off = np.abs(got - want) / (U * np.abs(want))
    assert (off <= e).all(), (off.max(), e[off.argmax()])
    w[at, at] = 0
    assert (w == 0).all()                                    # nothing beside the diagonal


@pytest.mark.parametrize("shape", [(64, 64), (100, 128), (128, 256), (64, 2000), (200, 200), (300, 500), (1024, 1024), (1511, 777), (999, 301), (1024, 4096)])
def test_random_matrices(d, shape):
    w, g, m = make(shape, 15)
    (nw, nm), = step(d, [(w, g, m)])
    # sums: half a step per cut on the average, 15 products of 24 * 2^-25 and 2^-22, twice (see the test of long sums): 2.9e-5.  X's own rounding, 2^-23 of |X| = 1,
    # grows by 3.4445^5 = 485 at most, against a result of |X| > 0.7 sqrt(side)
    close = 2.9e-5 + 485 * 2.0 ** -23 / (0.7 * min(shape) ** 0.5)
    assert close < CLOSE / 2
    check(nw, nm, w, g, m, close=close)
