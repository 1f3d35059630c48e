"""Pushes that name some rows very often, as the frequent words of a batch do:
M is mu M + g to the bit, g the f32 sum in the push's order."""
import numpy as np
import pytest
import torch

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def push(R, pushed, repeats, seed):
    """Rows of a push in any order: `repeats` of row -> times, the others
    from anywhere, outside the table among them."""
    g = torch.Generator().manual_seed(seed)
    rows = torch.randint(-3, R + 3, (pushed,), generator=g)
    at = torch.randperm(pushed, generator=g)
    for row, times in repeats.items():
        rows[rows == row] = -1
        rows[at[:times]] = row
        at = at[times:]
    return rows


def check(device, R, m, n, rows, sorted_first=False):
    g = torch.Generator().manual_seed(n)
    grads = torch.randn(rows.numel(), n, generator=g)
    mo = torch.randn(R, n, generator=g)
    if sorted_first:
        rows = rows.sort(stable=True).values
    total = np.zeros((R, n), dtype=np.float32)
    inside = (rows >= 0) & (rows < R)
    np.add.at(total, rows[inside].numpy(), grads[inside].numpy())
    named = torch.zeros(R // m, dtype=torch.bool)
    named[rows[inside] // m] = True
    want = torch.where(named.repeat_interleave(m)[:, None],
                       0.5 * mo + torch.from_numpy(total), mo)
    t, v = torch.zeros(R, n, device=device), mo.to(device)
    ops.apply_muon(t, v, rows.to(device), grads.to(device), 0.1, mu=0.5,
                   matrix_rows=m)
    assert torch.equal(v.cpu(), want)  # a product by 1/2 is exact
    assert torch.equal(t.cpu().view(R // m, -1).any(1), named)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 5, 16, 17, 33, 64, 65, 100, 130, 300])
@pytest.mark.parametrize("pushed", [2500, 17000])
def test_widths(device, n, pushed):
    rows = push(300, pushed, {0: 64, 7: 65, 8: 66, 100: 127, 101: 128,
                              102: 129, 200: 192, 201: 193, 298: 500,
                              299: 700}, n)
    check(device, 300, 300, n, rows)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("row", [0, 255, 256, 599, -1, 600])
@pytest.mark.parametrize("pushed", [65, 129, 16384, 16385])
def test_one_row(device, row, pushed):
    """All of a push for one row, inside the table or not."""
    check(device, 600, 200, 6, torch.full((pushed,), row))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("R,m,n,pushed", [
    (4000, 4000, 8, 16384), (3000, 3, 8, 16384), (3300, 3, 8, 9000),
    (64, 64, 20, 16000), (1000, 500, 520, 3000), (2000, 1000, 96, 16385),
    (4000, 2000, 40, 100000)])
def test_skewed(device, R, m, n, pushed):
    """A row's share of a push falls as its number rises."""
    g = torch.Generator().manual_seed(R + n)
    u = torch.rand(pushed, generator=g, dtype=torch.float64)
    rows = (torch.exp(u * np.log(R + 1.0)) - 1).long().clamp(max=R - 1)
    check(device, R, m, n, rows[torch.randperm(pushed, generator=g)])
    check(device, R, m, n, rows, sorted_first=True)


@pytest.mark.gpu
def test_replayed_with_other_repeats():
    R, n, pushed = 500, 24, 4000
    table, mo = (torch.randn(R, n, device="cuda") for _ in range(2))
    rows = push(R, pushed, {3: 900}, 0).cuda()
    grads = torch.randn(pushed, n, device="cuda")
    ops.apply_muon(table, mo, rows, grads, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.apply_muon(table, mo, rows, grads, 0.1)
    for k in range(4):
        rows.copy_(push(R, pushed, {k: 70 + k, 499: 1300 * k}, k))
        grads.copy_(torch.randn(pushed, n, device="cuda"))
        t, v = table.clone(), mo.clone()
        graph.replay()
        torch.cuda.synchronize()
        ops.apply_muon(t, v, rows, grads, 0.1)
        assert torch.equal(table, t) and torch.equal(mo, v)


@pytest.mark.gpu
def test_more_gradients_than_a_launch_has_blocks_for():
    """2^26 places are a launch's; ones are summed exactly below 2^24."""
    R, pushed = 700, 2 ** 26 + 12345
    rows = torch.randint(0, R - 1, (pushed,), device="cuda")
    rows[::7] = R - 1  # the last of the sorted ones: 9.6 million
    table, mo = (torch.zeros(R, 1, device="cuda") for _ in range(2))
    ops.apply_muon(table, mo, rows, torch.ones(pushed, 1, device="cuda"), 0.1)
    assert torch.equal(mo.view(-1).long(), torch.bincount(rows, minlength=R))


@pytest.mark.gpu
@pytest.mark.parametrize("R,n", [(3952, 32), (20000, 100), (2048, 512)])
def test_one_row_does_not_hold_up_a_step(R, n):
    """100,000 gradients of one row: a pass over them and a sort take a
    millisecond or two; one load after the other took 44 to 89."""
    table, mo = (torch.zeros(R, n, device="cuda") for _ in range(2))
    rows = torch.full((100000,), R // 2, device="cuda")
    grads = torch.randn(100000, n, device="cuda")
    took = []
    for _ in range(4):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        ops.apply_muon(table, mo, rows, grads, 0.1)
        end.record()
        torch.cuda.synchronize()
        took.append(begin.elapsed_time(end))
    assert min(took) <= 15
