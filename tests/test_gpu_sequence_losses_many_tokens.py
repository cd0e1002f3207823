"""The losses over packed sequences of more tokens than a CTA for each SM has: the policy loss takes two parts to a CTA above 303104 tokens, sums its CTAs by a
kernel of its own above 2097152, and counts its tokens by one above 8388608."""
import pytest

import __graft_entry__ as ge

ge.load_package()
from test_gpu_sequence_losses import batch, check, policy, preference  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


@pytest.mark.parametrize("tokens,sequences", [(303104, 40), (303105, 40), (700001, 9), (2097152, 300), (2097153, 100000), (2300000, 1)])
@pytest.mark.parametrize("by_sequence", [False, True])
@pytest.mark.parametrize("per_token", [False, True])
def test_policy_loss(d, tokens, sequences, by_sequence, per_token):
    check(policy(d, batch(80, tokens, sequences, before=5, behind=777), per_token=per_token, by_sequence=by_sequence))


@pytest.mark.parametrize("kind,by_sequence,per_token,reference,shift", [("f32", False, False, True, 0), ("i64", False, True, False, 1), ("i32", True, False, True, 0)])
@pytest.mark.parametrize("tokens", [8388608, 8388609, 8700000])
def test_policy_loss_of_more_tiles_than_a_cta_adds_up(d, tokens, kind, by_sequence, per_token, reference, shift):
    check(policy(d, batch(81, tokens, 4000, before=1, behind=3001), kind=kind, per_token=per_token, by_sequence=by_sequence, reference=reference, entropy=False,
                 shift=shift), entropy=False)


def test_policy_loss_of_a_larger_batch_and_without_gradients(d):
    b = batch(82, 8500001, 33)
    check(policy(d, b, per_token=False, count=1e7, gradient=False, entropy=False), gradient=False, entropy=False)


@pytest.mark.parametrize("tokens,pairs,kind,average", [(4500001, 40, "i32", True), (8400000, 3, "f32", False), (3000000, 100000, "i64", True)])
def test_loss_of_pairs(d, tokens, pairs, kind, average):
    preference(d, batch(83, tokens, 2 * pairs, before=9, behind=1234), kind=kind, average=average, smoothing=0.1)
