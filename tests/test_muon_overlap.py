"""apply_muon on operands that lie in one piece of memory."""
import pytest
import torch

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shift", [0, 1, 7, 59])
def test_table_and_momentum_must_not_overlap(device, shift):
    both = torch.ones(60 + shift, 8, device=device)
    before = both.clone()
    rows = torch.arange(60, device=device)
    grads = torch.ones(60, 8, device=device)
    for table, mo in ((both[:60], both[shift:]), (both[shift:], both[:60])):
        with pytest.raises(ValueError, match="same memory"):
            ops.apply_muon(table, mo, rows, grads, 0.1)
    assert torch.equal(both, before)
    # side by side they are two
    ops.apply_muon(torch.ones(120, 8, device=device)[:60],
                   torch.ones(120, 8, device=device)[60:], rows, grads, 0.1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", [(30, 8), (300, 100), (150, 200)])
@pytest.mark.parametrize("which", ["table", "momentum"])
def test_gradients_in_the_memory_of_a_table(device, which, m, n):
    """They are read as they were before the step, in any order."""
    g = torch.Generator().manual_seed(m)
    table, mo = (torch.randn(2 * m, n, generator=g).to(device)
                 for _ in range(2))
    rows = torch.randperm(2 * m, generator=g).to(device)
    apart = [table.clone(), mo.clone()]
    grads = table if which == "table" else mo
    ops.apply_muon(*apart, rows, grads.clone(), 0.1, matrix_rows=m)
    ops.apply_muon(table, mo, rows, grads, 0.1, matrix_rows=m)
    assert torch.equal(table, apart[0]) and torch.equal(mo, apart[1])
