"""The kernels that the operators around drafted tokens say they launched, against the kernel nodes of a recorded graph."""
import numpy as np
import pytest
import torch

from safetyraise_lmengine_b200.kernels import ops
from test_drafts_gpu import DEV, Case, ints

pytestmark = pytest.mark.gpu


def counted(call):
    """(what ops.launches grew by, kernels that a graph of the call holds)."""
    from cuda.bindings import runtime as rt
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        before = ops.launches
        call()
        grown = ops.launches - before
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    n = rt.cudaGraphGetNodes(raw)[-1]
    nodes = rt.cudaGraphGetNodes(raw, n)[1]
    kernels = sum(rt.cudaGraphNodeGetType(node)[1] == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for node in nodes)
    return grown, kernels


@pytest.mark.parametrize("dt, hd, ps", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 20), (torch.float32, 64, 16)])
@pytest.mark.parametrize("n, ctx, both", [(1, 30, 1), (1, 3000, 2), (40, 30, 2)])
def test_attention(dt, hd, ps, n, ctx, both):
    """One kernel where no unit is divided, else a second one that adds what several blocks have."""
    c = Case([3] * n, [ctx] * n, 8, 2, hd, ps, dt)
    assert counted(c.run) == (both, both)


def test_the_others():
    pool = torch.zeros(2, 2200, 1, 4, 8, device=DEV)
    for pages in (1, 16, 17, 480, 481, 1000):
        src, dst = list(range(pages)), list(range(1100, 1100 + pages))
        want = -(-pages // 480)
        assert counted(lambda: ops.copy_pages(pool, src, dst)) == (want, want), pages
    positions, mask, cu, kv = ints([0] * 3), ints(np.zeros((3, 1))), ints([0, 3]), ints([5])
    parents, path, count, nxt = ints([-1, 0, 1]), ints([[0] * 3]), ints([0]), ints([0])
    table = ints([[0, 1]])
    assert counted(lambda: ops.draft_tree(parents, cu, kv, positions, mask)) == (1, 1)
    assert counted(lambda: ops.accept_drafts(parents, parents, parents, cu, path, count, nxt)) == (1, 1)
    assert counted(lambda: ops.keep_drafts(pool, table, cu, kv, path, count)) == (1, 1)


def test_what_launches_nothing_counts_nothing():
    pool = torch.zeros(2, 4, 1, 4, 8, device=DEV)
    before = ops.launches
    ops.copy_pages(pool, [], [])
    ops.draft_tree(ints([]), ints([0]), ints([]), ints([]), ints(np.zeros((0, 1))))
    assert ops.launches == before
