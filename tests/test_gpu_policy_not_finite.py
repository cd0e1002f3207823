"""The policy loss where its inputs are not finite, or a term's value is too large for fp32 but its weight zero."""
import math

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from test_gpu_sequence_losses import batch, policy  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


# one CTA, two or three kernels
@pytest.mark.parametrize("tokens", [500, 30000])
@pytest.mark.parametrize("per_token", [True, False])
@pytest.mark.parametrize("by_sequence", [True, False])
@pytest.mark.parametrize("difference", [0.5, -0.5, math.log1p(float(np.float32(0.25)))])
def test_an_advantage_that_is_none_shows_in_the_gradient(d, tokens, per_token, by_sequence, difference):
    b = batch(60, tokens, 9, empty_rows=False)
    first, last = (int(v) for v in b["offsets"][3:5])
    assert last - first > 10
    # tokens whose ratio is past a border, or on one: with a number for an advantage they may count as clipped
    b["old"][first:last] = b["logprob"][first:last] - np.float32(difference)
    counts = (b["ids"] >= 0) & (np.arange(tokens) >= first) & (np.arange(tokens) < last)
    bad = np.zeros(tokens, bool)
    if per_token:
        bad[np.flatnonzero(counts)[:3]] = True
        b["token_advantage"][bad] = math.nan
    else:
        bad, b["advantage"][3] = counts, math.nan
    loss, g, h, (want, wg, _, _) = policy(d, b, per_token=per_token, by_sequence=by_sequence)
    assert np.isnan(wg[bad]).all() and np.isfinite(wg[~bad]).all()
    assert np.isnan(g[bad]).all() and np.isfinite(g[~bad]).all() and np.isfinite(h).all()
    assert np.isnan(loss[:2]).all() and np.isfinite(loss[2:]).all()
    assert abs(loss[4] - want[4]) <= 1e-6                    # (shares of a few hundred tokens, summed in fp32) none of them is clipped
