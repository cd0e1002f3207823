"""A term of the policy loss whose weight is zero is no part of the loss nor of its gradients, whatever the term itself comes to."""
import math

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
from test_gpu_sequence_losses import batch, check, policy  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


@pytest.mark.parametrize("tokens", [500, 30000])
@pytest.mark.parametrize("by_sequence", [True, False])
@pytest.mark.parametrize("far", [100.0, 1e4, math.inf, math.nan])
def test_a_term_of_weight_zero_is_left_out(d, tokens, by_sequence, far):
    b = batch(61, tokens, 9)
    without = policy(d, b, reference=False, entropy=False, by_sequence=by_sequence)
    check(without, entropy=False)
    # references that the policy has moved far away from: exp(100) is beyond fp32
    b["reference"] = (b["logprob"] + np.float32(far)).astype(np.float32)
    b["entropy"][:] = far if far > 1e4 else 1.0
    loss, g, h, _ = policy(d, b, by_sequence=by_sequence, kl_weight=0.0, entropy_weight=0.0)
    assert loss[0] == without[0][0] and loss[1] == without[0][1] and loss[4] == without[0][4]
    assert np.array_equal(g, without[1]) and (h == 0).all()
    assert not np.isfinite(loss[2])                          # its mean is reported all the same
