"""What a step of orthogonalised momentum does when a wait on the device has given up: the products that follow have no operands that mean
anything, and the last ones leave the weights alone.  The word that says so, first in the workspace, is set by a node that is put into the captured step."""
import ctypes

import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from polarai_framework_b200.capi import MuonOptions, MuonTensor  # noqa: E402
from test_gpu_muon import A, B, C, check, make  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def ok(result):
    error, *rest = result
    assert int(error) == 0, error
    return rest[0] if len(rest) == 1 else rest


# short sums shared by clusters, tiles of 128 and of 256 columns, narrow matrices, several of them and odd sizes that are not read as vectors
@pytest.mark.parametrize("shapes", [[(300, 200)], [(1024, 1024)], [(2048, 4096)], [(90, 2000)], [(301, 257), (700, 300)], [(3, 200, 1000), (40, 600)]])
@pytest.mark.parametrize("failed", [0, 1])
def test_weights_stay_when_a_wait_has_given_up(d, shapes, failed):
    from cuda.bindings import runtime
    ts = [make(s, 40 + i) for i, s in enumerate(shapes)]
    new = [(w.clone(), m.clone()) for w, _, m in ts]
    arr = (MuonTensor * len(ts))()
    for t, (w, m), (_, g, _) in zip(arr, new, ts):
        t.weights, t.gradient, t.momentum = w.data_ptr(), g.data_ptr(), m.data_ptr()
        t.rows, t.cols = w.shape[-2:]
        t.matrices, t.scale = w.numel() // (t.rows * t.cols), max(1.0, t.rows / t.cols) ** 0.5
    options = MuonOptions(0.5, 0.95, 1, 5, A, B, C, None)
    need = d.lib.cdll.polar_b200_fmuon_workspace_bytes(arr, len(ts))
    workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    call = lambda: d.lib.call("polar_b200_fmuon", arr, len(ts), ctypes.byref(options), workspace.data_ptr(), need,  # noqa: E731
                              torch.cuda.current_stream().cuda_stream)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    raw = runtime.cudaGraph_t(graph.raw_cuda_graph())
    count = ok(runtime.cudaGraphGetNodes(raw))[1]
    nodes = ok(runtime.cudaGraphGetNodes(raw, count))[0]
    assert count >= 8                                        # two passes, a product or more for each round
    params = runtime.cudaMemsetParams()
    params.dst, params.elementSize, params.width, params.height, params.value, params.pitch = workspace.data_ptr(), 4, 1, 1, failed, 0
    # behind the two passes and before the first product: a short list's last product comes before the graph's last node
    node = ok(runtime.cudaGraphAddMemsetNode(raw, [nodes[1]], 1, params))
    ok(runtime.cudaGraphAddDependencies(raw, [node], [nodes[2]], 1))
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    assert d.device_status() == 0
    for (w, m), t in zip(new, ts):
        if failed:
            assert torch.equal(w, t[0])
        else:
            check(w, m, *t)
    # the next step is a whole one again
    for (w, m), t in zip(new, ts):
        w.copy_(t[0]), m.copy_(t[2])
    call()
    torch.cuda.synchronize()
    for n, t in zip(new, ts):
        check(*n, *t)
