"""fadamw over as many tensors as its tables of the tensors' places hold, one less and one more; tensors of several chunks at a table's ends."""
import pytest

from test_gpu_adamw import check, env, make, step_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("count", [15, 16, 17, 63, 65, 129, 191, 192, 193, 447, 448, 449])
def test_counts_of_tensors(env, count, eight):  # noqa: F811
    torch, d = env
    sizes = [1 + (i * 7919) % 3000 for i in range(count)]
    # a chunk is 1024 or 2048 weights: several of them first and last, in the middle, and where the tables of 16, 192 and 448 tensors end
    for i in (0, 7, 8, 15, 63, 64, 127, 128, 191, 192, 383, 384, 447, 448, count - 1):
        if i < count:
            sizes[i] = 6145 + 128 * (i % 5)
    pairs = [make(torch, n, eight, seed=i) for i, n in enumerate(sizes)]
    decays = [0.05 * (i % 4) for i in range(count)]
    step_of(d, [p[1] for p in pairs], eight, step=5, lr=2e-3, weight_decay=decays)
    for (host, dev), n, decay in zip(pairs, sizes, decays):
        check(torch, host, dev, n, eight, 5, lr=2e-3, decay=decay)


@pytest.mark.parametrize("eight", [False, True])
def test_tensors_in_descending_order_in_memory(env, eight):  # noqa: F811
    # neither order of the arrays in memory nor of the list changes a bit
    torch, d = env
    pairs = [make(torch, 500 + 37 * i, eight, seed=i) for i in range(40)]
    again = [{k: v.clone() for k, v in p[1].items()} for p in pairs]
    step_of(d, [p[1] for p in pairs], eight, step=3, lr=1e-3)
    step_of(d, again[::-1], eight, step=3, lr=1e-3)
    for (_, dev), other in zip(pairs, again):
        assert all(torch.equal(dev[k], other[k]) for k in dev)
