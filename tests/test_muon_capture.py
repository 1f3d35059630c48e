"""Which pushes in any order a captured graph takes, by what is refused."""
import pytest
import torch

from flink_parameter_server_amd import ops


@pytest.mark.gpu
@pytest.mark.parametrize("matrices,m,taken", [
    (2 ** 20, 1, True), (2 ** 20 + 1, 1, False), (2 ** 19, 257, True),
    (2 ** 19 + 1, 257, False)])
def test_windows(matrices, m, taken):
    """A matrix of 257 rows has two windows."""
    table = torch.zeros(matrices * m, 1, device="cuda")
    mo = torch.zeros_like(table)
    rows = torch.tensor([5, 0, table.shape[0] - 1], device="cuda")
    grads = torch.ones(3, 1, device="cuda")
    one = torch.zeros(8, device="cuda")
    ops.apply_muon(table, mo, rows, grads, 0.0, matrix_rows=m)
    mo.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one += 1  # the graph has a node
        if taken:
            ops.apply_muon(table, mo, rows, grads, 0.0, matrix_rows=m)
        else:
            with pytest.raises(RuntimeError, match="windows .256 rows"):
                ops.apply_muon(table, mo, rows, grads, 0.0, matrix_rows=m)
    for k in range(3):
        mo.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert float(mo.sum()) == (3.0 if taken else 0.0)
        assert bool((one == k + 1).all())
