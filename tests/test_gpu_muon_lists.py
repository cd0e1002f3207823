"""Orthogonalised momentum over lists whose matrices need different numbers of products, against the formula in 64 bits."""
import pytest

import __graft_entry__ as ge

ge.load_package()
from test_gpu_muon import check, make, step  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("shapes", [[(777, 611), (500, 170), (150, 257)], [(512, 512), (256, 512)], [(300, 290), (140, 290), (700, 10)], [(400, 260), (300, 100)]])
def test_the_first_matrix_has_the_shorter_list_of_products(d, shapes, steps):
    # the longest side comes first: within a factor of two of the other one, three products a round; the others take seven for two rounds
    ts = [make(s, 30 + i) for i, s in enumerate(shapes)]
    for (nw, nm), t in zip(step(d, ts, steps=steps), ts):
        check(nw, nm, *t, steps=steps)
