"""A server table that steps with Muon under several workers: a round's pushes
are one step of the matrices that they name rows of."""
import pytest
import torch

from flink_parameter_server_amd import (PSConfig, PSEngine, RangePartitioner,
                                        ShardedTable, TableServerLogic,
                                        WorkerLogic, ops)
from flink_parameter_server_amd.parallel.transport import run_loopback

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
FEEDBACKS = ["fresh", "merged", "pipelined"]
COUNT, M, N = 4, 12, 7  # matrices of a job's table, rows and columns of each
LR, DECAY = 0.1, 0.02


class Pushes(WorkerLogic):
    """Pushes what it is given, without a pull."""

    def on_recv(self, data, client):
        client.push(*data)

    def on_pull_recv(self, ids, values, client):
        raise AssertionError("nothing was pulled")


def train(world, data, device, feedback, unique=True, **config):
    """The tables and momenta after ``data[rank]`` (a list of pushes) went
    through ``world`` ranks, a shard each."""
    def job(rank, transport):
        part = RangePartitioner(COUNT * M, world)
        table = ShardedTable(part, rank, N, device, init=(-0.5, 0.5),
                             optimizer="muon", lr=LR, weight_decay=DECAY,
                             matrix_rows=M)
        engine = PSEngine(
            PSConfig(num_ids=COUNT * M, dim=N, partitioner="range",
                     feedback=feedback, **config), Pushes(),
            TableServerLogic(table, dump_on_close=False,
                             pushes_unique=unique),
            transport, part, device=device)
        engine.run(data[rank])
        return table.data, table.accum
    tables, momenta = zip(*run_loopback(world, job))
    return torch.cat(tables), torch.cat(momenta)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("feedback", FEEDBACKS)
@pytest.mark.parametrize("world", [2, 4])
def test_shares_of_a_gradient_make_its_step(device, feedback, world):
    """Workers that push g / W each leave what one that pushes g leaves, to
    the bit: W is a power of two, so that the shares' sum is g."""
    g = torch.Generator().manual_seed(world)
    ids = torch.arange(COUNT * M, device=device)
    grads = [torch.randn(COUNT * M, N, generator=g).to(device)
             for _ in range(3)]
    alone = train(world, [[(ids, v) for v in grads]] + [[]] * (world - 1),
                  device, feedback)
    shared = train(world, [[(ids, v / world) for v in grads]] * world, device,
                   feedback)
    assert torch.equal(shared[0], alone[0])
    assert torch.equal(shared[1], alone[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("feedback", FEEDBACKS)
def test_a_round_is_the_step_of_its_joined_pushes(device, feedback):
    """Different rows of each worker, some of them in common, matrices that
    one worker or nobody names: the tables equal calls of ``apply_muon`` with
    the pushes one after the other in rank order."""
    g = torch.Generator().manual_seed(8)
    half = COUNT * M // 2
    rows = [torch.tensor([0, 1, 5, 11, 25, 30]), torch.tensor([1, 2, 5, 40]),
            None, torch.tensor([3, 11])]
    pushes = [None if r is None else
              (r.to(device),
               torch.randn(r.numel(), N, generator=g).to(device))
              for r in rows]
    # two shards of two matrices: the other two ranks have workers alone
    def job(rank, transport):
        part = RangePartitioner(COUNT * M, 2)
        table = ShardedTable(part, rank, N, device, init=(-0.5, 0.5),
                             optimizer="muon", lr=LR, weight_decay=DECAY,
                             matrix_rows=M) if rank < 2 else None
        start = None if table is None else table.data.clone()
        engine = PSEngine(
            PSConfig(n_workers=4, n_shards=2, num_ids=COUNT * M, dim=N,
                     partitioner="range", feedback=feedback), Pushes(),
            TableServerLogic(table, dump_on_close=False, pushes_unique=True),
            transport, part, device=device)
        engine.run([] if pushes[rank] is None else [pushes[rank]])
        return table and (start, table.data, table.accum)
    shards = run_loopback(4, job)
    for k in range(2):
        start, data, accum = shards[k]
        mine = [((r >= k * half) & (r < (k + 1) * half), r, v)
                for r, v in (p for p in pushes if p is not None)]
        momentum = torch.zeros_like(start)
        ops.apply_muon(start, momentum,
                       torch.cat([r[at] - k * half for at, r, _ in mine]),
                       torch.cat([v[at] for at, _, v in mine]), LR,
                       weight_decay=DECAY, matrix_rows=M)
        assert torch.equal(data, start) and torch.equal(accum, momentum)


@pytest.mark.parametrize("optimizer", ["add", "adagrad"])
def test_other_rules_take_pushes_one_by_one(optimizer):
    """A subclass sees what every worker pushed, as before."""
    class Seen(TableServerLogic):
        def on_push_recv(self, ids, deltas, ps):
            self.seen.append((ids.tolist(), self.pushes_unique))
            super().on_push_recv(ids, deltas, ps)

    def job(rank, transport):
        part = RangePartitioner(8, 2)
        logic = Seen(ShardedTable(part, rank, 2, "cpu", optimizer=optimizer,
                                  lr=0.1), pushes_unique=True)
        logic.seen = []
        PSEngine(PSConfig(num_ids=8, dim=2, partitioner="range"), Pushes(),
                 logic, transport, part).run(
            [(torch.tensor([1, 3 + rank, 6]), torch.ones(3, 2))])
        return logic.seen
    assert run_loopback(2, job) == [
        [([1, 3], True), ([1], True)], [([6], True), ([4, 6], True)]]


def test_a_muon_server_refuses_a_pull_limit():
    part = RangePartitioner(2 * M, 1)
    server = TableServerLogic(ShardedTable(part, 0, N, "cpu",
                                           optimizer="muon", lr=LR))
    with pytest.raises(ValueError, match="pull limit"):
        PSEngine(PSConfig(num_ids=2 * M, dim=N, partitioner="range",
                          pull_limit=M), Pushes(), server, None, part)
    limited = Pushes()
    limited.pull_limit = 3
    with pytest.raises(ValueError, match="pull limit"):
        PSEngine(PSConfig(num_ids=2 * M, dim=N, partitioner="range"),
                 limited, server, None, part)
    plain = TableServerLogic(ShardedTable(part, 0, N, "cpu"))
    PSEngine(PSConfig(num_ids=2 * M, dim=N, partitioner="range",
                      pull_limit=M), Pushes(), plain, None, part)
