"""GPU tests of the small-batch GEMMs' plans: the grid of a call, read from a captured
graph."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def ok(result):
    err, *values = result
    assert int(err) == 0, err
    return values[0] if len(values) == 1 else values


def captured_kernels(call):
    """(kernel node, parameters, CTAs of a cluster) of every kernel that `call` launches."""
    driver = pytest.importorskip("cuda.bindings.driver")
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    graph = driver.CUgraph(g.raw_cuda_graph())
    nodes, count = ok(driver.cuGraphGetNodes(graph))
    nodes, count = ok(driver.cuGraphGetNodes(graph, count))
    found = []
    for node in nodes[:count]:
        if ok(driver.cuGraphNodeGetType(node)) != driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        params = ok(driver.cuGraphKernelNodeGetParams(node))
        value = ok(driver.cuGraphKernelNodeGetAttribute(
            node, driver.CUkernelNodeAttrID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION))
        found.append((driver, params, max(value.clusterDim.x, 1)))
    return g, found


def resident(driver, params, cluster):
    """Clusters of the launch that fit on the GPU at once."""
    cfg = driver.CUlaunchConfig()
    cfg.gridDimX, cfg.gridDimY, cfg.gridDimZ = cluster, 1, 1
    cfg.blockDimX, cfg.blockDimY, cfg.blockDimZ = params.blockDimX, params.blockDimY, params.blockDimZ
    cfg.sharedMemBytes = params.sharedMemBytes
    attr = driver.CUlaunchAttribute()
    attr.id = driver.CUlaunchAttributeID.CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION
    attr.value.clusterDim.x, attr.value.clusterDim.y, attr.value.clusterDim.z = cluster, 1, 1
    cfg.attrs, cfg.numAttrs = [attr], 1
    func = params.func
    if int(func) == 0:  # the node names a context-independent kernel
        func = ok(driver.cuKernelGetFunction(params.kern))
    return ok(driver.cuOccupancyMaxActiveClusters(func, cfg))


# tiles of 64 to 256 columns in slices of three and four: near as many CTAs as SMs
@pytest.mark.parametrize("N", [1024, 1056, 1088, 1152, 1184, 1440, 1536, 2304, 2368, 2816, 2880, 4096, 4320, 4608,
                               5632, 5760, 6016, 6144, 9472])
@pytest.mark.parametrize("M,K", [(1, 4096), (101, 2048)])
def test_slices_of_a_gated_gemm_are_resident_together(M, K, N):
    from evo2_flash_b200 import ops

    x = torch.zeros(M, K, dtype=BF, device=DEV)
    w1, w2 = (torch.zeros(N, K, dtype=BF, device=DEV) for _ in range(2))
    graph, kernels = captured_kernels(lambda: ops.gemm_gated_bf16(x, w1, w2))
    assert len(kernels) == 1
    driver, params, cluster = kernels[0]
    if cluster > 1:
        assert cluster == params.gridDimX
        assert params.gridDimY <= resident(driver, params, cluster)
    del graph
