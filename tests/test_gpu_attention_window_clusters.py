"""GPU: windowed attention, forward: where the CTAs of a cluster share a unit's keys, the device seats all clusters of the launch at once. A
cluster lies within one GPC, so that fewer of them find a place than the SMs would hold, and those left over would run after the others."""
import pytest

pytestmark = pytest.mark.gpu


def _launches(call):
    """(clusters, CTAs of a cluster, clusters that the device seats at once) of every kernel that `call` launches, from a captured graph."""
    import torch
    from cuda.bindings import driver as cu

    def ok(r):
        assert r[0] == cu.CUresult.CUDA_SUCCESS, r[0]
        return r[1] if len(r) == 2 else r[1:]

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw, out = cu.CUgraph(graph.raw_cuda_graph()), []
    n = ok(cu.cuGraphGetNodes(raw))[1]
    for node in ok(cu.cuGraphGetNodes(raw, n))[0][:n]:
        if ok(cu.cuGraphNodeGetType(node)) != cu.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        k = ok(cu.cuGraphKernelNodeGetParams(node))
        size = ok(cu.cuGraphKernelNodeGetAttribute(node, cu.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION)).clusterDim.x
        if size <= 1:
            continue
        c, a = cu.CUlaunchConfig(), cu.CUlaunchAttribute()
        a.id = cu.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION
        a.value.clusterDim.x, a.value.clusterDim.y, a.value.clusterDim.z = size, 1, 1
        c.gridDimX, c.gridDimY, c.gridDimZ, c.blockDimX, c.blockDimY, c.blockDimZ = k.gridDimX, 1, 1, k.blockDimX, 1, 1
        c.sharedMemBytes, c.attrs, c.numAttrs = k.sharedMemBytes, [a], 1
        out.append((k.gridDimX // size, size, ok(cu.cuOccupancyMaxActiveClusters(k.func, c))))
    return out


def _forward(q_lens, k_lens, hq, hkv, hd, window):
    import torch

    from ml_dataflow_b200 import ops

    offs = lambda lens: [sum(lens[:i]) for i in range(len(lens))]
    rand = lambda n, c: torch.randn((n, c), device="cuda").to(torch.bfloat16)
    q, k, v = rand(sum(q_lens), hq * hd), rand(sum(k_lens), hkv * hd), rand(sum(k_lens), hkv * hd)
    o, lse = torch.empty_like(q), torch.empty((hq, sum(q_lens)), device="cuda")
    return lambda: ops.attention_window_fwd(offs(q_lens), q_lens, offs(k_lens), k_lens, hq, hkv, hd, q, k, v, o, lse, window, 0)


@pytest.mark.parametrize("hd", [128, 64])
def test_tiles(hd):
    from gpu_util import require_b200

    require_b200()
    sizes = set()
    for pairs in range(1, 76):
        for blocks in (10, 24):
            call = _forward([128 * pairs], [128 * (pairs + blocks)], 2, 1, hd, 128 * (blocks - 2))
            call()
            for clusters, size, seats in _launches(call):
                assert clusters == pairs <= seats, (pairs, blocks, size, seats)
                sizes.add(size)
    assert sizes == {2, 4, 8}


@pytest.mark.parametrize("hd", [128, 64])
def test_few_queries(hd):
    from gpu_util import require_b200

    require_b200()
    sizes = set()
    for units in range(1, 160):
        call = _forward([1] * units, [1200] * units, 4, 1, hd, 1000)
        call()
        for clusters, size, seats in _launches(call):
            assert clusters == units <= seats, (units, size, seats)
            sizes.add(size)
    assert sizes == {2, 4, 8}
