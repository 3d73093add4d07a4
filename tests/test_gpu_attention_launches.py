"""What a gradient call launches: a grid that overlaps the one before it sees what came earlier only if it waits itself,
so that the split of the operands has to stand directly in front of the one launch that reads it."""
import ctypes as C

import pytest

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu

KERNEL = 0  # CU_GRAPH_NODE_TYPE_KERNEL


def kernels_of(dev, call):
    """Kernel nodes of a captured call."""
    t, cu = dev.torch, C.CDLL("libcuda.so.1")
    graph = t.cuda.CUDAGraph(keep_graph=True)
    with t.cuda.graph(graph):
        call(t.cuda.current_stream().cuda_stream)
    g, count = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert cu.cuGraphGetNodes(g, None, C.byref(count)) == 0
    nodes = (C.c_void_p * count.value)()
    assert cu.cuGraphGetNodes(g, nodes, C.byref(count)) == 0
    kinds = {}
    for n in nodes:
        kind = C.c_int(-1)
        assert cu.cuGraphNodeGetType(C.c_void_p(n), C.byref(kind)) == 0
        kinds[n] = kind.value
    return [n for n in nodes if kinds[n] == KERNEL]


@pytest.mark.parametrize("heads,kv_heads,n,launches", [(32, 32, 2000, 2), (2, 1, 3000, 3)])
def test_launches_of_a_gradient(jx, dev, heads, kv_heads, n, launches):
    """The split and the gradients; the sum of the parts where key tiles are few, which nothing overlaps."""
    c = Case(dev, [n], [n], heads, kv_heads, 64)
    c.forward(jx)
    c.backward(jx)
    dev.sync()
    assert len(kernels_of(dev, lambda st: c.backward(jx, stream=st))) == launches
