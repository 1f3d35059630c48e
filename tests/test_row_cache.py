"""8-bit row records (ops.cache_write / ops.cache_read): the records against
a 64-bit implementation written from the format's definition, the HIP kernels
against the oracle byte for byte, refusals, and the wire that carries them.

No tolerances but one: codes and scales are those of exactly rounded
operations, so records and values have to be equal.  What a value may be off
its original by is the format's own: half a step of the row for int8
(amax / 254), half a step of e4m3 for fp8 (2^-4 relative; 2^-10 scales below
2^-6 scales, where e4m3 is subnormal).
"""
import math

import pytest
import torch

from flink_parameter_server_amd import PSConfig, PSEngine, ops
from flink_parameter_server_amd import (ModPartitioner, ShardedTable,
                                        TableServerLogic, WorkerLogic)
from flink_parameter_server_amd.ops import reference as R
from flink_parameter_server_amd.parallel.transport import run_loopback

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
FORMATS = ["int8", "fp8"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
BIG = 3.4028234663852886e38
TINY = 2.0 ** -126


def e4m3_values():
    out = []
    for k in range(127):
        e, f = divmod(k, 8)
        out.append(f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10))
    return torch.tensor(out, dtype=torch.float64)


def definition(x, fmt):
    """(codes as bytes, scale) of the rows of x, row by row in 64 bits."""
    codes, scales = [], []
    table = e4m3_values()
    for row in x.double():
        if not bool(torch.isfinite(row).all()):
            codes.append(torch.zeros(row.numel(), dtype=torch.uint8))
            scales.append(float("nan"))
            continue
        amax = float(row.abs().max())
        if fmt == "int8":
            # f32 nearest to the exact quotient (53 bits hold it closely
            # enough: no 24-bit value over 127 lies that near to a half step)
            s = max(float(torch.tensor(amax / 127, dtype=torch.float32)),
                    TINY)
            while 127 * s > BIG:  # the largest code has to be finite
                s = float(torch.nextafter(torch.tensor(s), torch.tensor(0.)))
            q = [round(float(v) / s) for v in row]  # ties to even
            codes.append(torch.tensor([v % 256 for v in q],
                                      dtype=torch.uint8))
        else:
            s = TINY
            while amax > 448 * s:
                s *= 2
            q = []
            top = 240 * 2.0 ** 120  # the next value up is 2^128
            for v in row.clamp(-top, top).tolist():
                d = (table - abs(v) / s).abs()
                best = torch.nonzero(d == d.min()).reshape(-1).tolist()
                c = best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1]
                q.append(c + (128 if math.copysign(1, v) < 0 else 0))
            codes.append(torch.tensor(q, dtype=torch.uint8))
        scales.append(s)
    return torch.stack(codes), torch.tensor(scales, dtype=torch.float32)


def awkward_rows(dim, g):
    """Rows where rounding goes wrong first."""
    rows = [torch.zeros(dim), torch.full((dim,), -3.0),
            torch.randn(dim, generator=g) * 1e-30,
            torch.randn(dim, generator=g) * 2.0 ** -140,   # subnormal
            torch.full((dim,), 2.0 ** -149),
            torch.randn(dim, generator=g).clamp(-1, 1) * 3e38,
            torch.full((dim,), BIG)]
    # halves of int8 steps (scale 1 and 0.37), and the largest code
    half = torch.randint(-126, 126, (dim,), generator=g) + 0.5
    half[0] = 127.0
    rows += [half, half * 0.37, half * 2.0 ** 90]
    # middles of e4m3 neighbours under scale 1, and its borders
    t = e4m3_values().float()
    mid = ((t[1:] + t[:-1]) / 2)[torch.randint(0, 126, (dim,), generator=g)]
    mid[0] = 448.0
    rows += [mid, -mid]
    for top in (448.0, 448.00003, 449.0, 224.0, 256.0, 1.75, 1.7500001):
        r = torch.randn(dim, generator=g).clamp(-1, 1) * top
        r[-1] = top
        rows.append(r)
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.randn(dim, generator=g)
        r[dim // 2] = bad
        rows.append(r)
    r = torch.randn(dim, generator=g)
    r[0], r[-1] = float("inf"), float("nan")
    rows.append(r)
    return torch.stack(rows)


def split(cache, dim):
    return cache[:, :dim].cpu(), cache[:, -4:].contiguous().cpu().view(
        torch.float32).reshape(-1)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=123.25),
                       torch.nan_to_num(b, nan=123.25)) and \
        torch.equal(torch.isnan(a), torch.isnan(b))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 31, 77])
def test_records_are_the_definition(device, fmt, dim):
    g = torch.Generator().manual_seed(dim)
    x = torch.cat([awkward_rows(dim, g), torch.randn(20, dim, generator=g)])
    cache = torch.full((x.shape[0], ops.record_bytes(dim)), 255,
                       dtype=torch.uint8, device=device)
    ops.cache_write(cache, x.to(device), fmt=fmt)
    codes, scales = split(cache, dim)
    want_codes, want_scales = definition(x, fmt)
    assert same(scales, want_scales)
    zero = want_codes % 128 == 0 if fmt == "fp8" else want_codes == 0
    # -0.0 and what rounds to it may keep its sign or not
    assert torch.equal(torch.where(zero & (codes % 128 == 0),
                                   want_codes, codes), want_codes)
    assert int(cache[:, dim:-4].cpu().sum()) == 0
    back = ops.cache_read(cache, dim, fmt=fmt).cpu()
    if fmt == "int8":
        values = torch.where(codes > 127, codes.double() - 256,
                             codes.double())
    else:
        values = e4m3_values()[(codes % 128).long()] * torch.where(
            codes > 127, -1.0, 1.0)
    want = values * scales.double()[:, None]
    assert same(back, want.float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_largest_values_stay_finite(device, fmt):
    x = torch.tensor([[BIG, -BIG, BIG / 2], [1.7e38, 1.0, -1.0]],
                     device=device)
    cache = ops.row_cache(2, 3, device)
    ops.cache_write(cache, x, fmt=fmt)
    assert bool(torch.isfinite(ops.cache_read(cache, 3, fmt=fmt)).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_distance_from_the_values(device, fmt):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 33, generator=g) * torch.exp(
        3 * torch.randn(500, 1, generator=g))
    cache = ops.row_cache(500, 33, device)
    ops.cache_write(cache, x.to(device), fmt=fmt)
    back = ops.cache_read(cache, 33, fmt=fmt).cpu().double()
    x = x.double()
    amax = x.abs().amax(1, keepdim=True)
    if fmt == "int8":
        # half a step, and the roundings of scale and product: 127.5 steps
        # of 2^-24 relative each
        limit = amax / 254 + 2 * amax * 2.0 ** -24
    else:
        # a scale is at most amax / 224
        limit = torch.maximum(x.abs() * 2.0 ** -4, amax / 224 * 2.0 ** -10)
    assert bool(((back - x).abs() <= limit).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (1, 128), (7, 300), (1000, 32),
                                   (64, 1025), (3, 5000), (2, 40000)])
def test_types_and_sizes_match_the_oracle(device, fmt, dtype, n, dim):
    g = torch.Generator().manual_seed(n + dim)
    x = (torch.randn(n, dim, generator=g)).to(dtype)
    want = ops.row_cache(n, dim)
    R.cache_write(want, x, fmt=fmt)
    cache = ops.row_cache(n, dim, device)
    ops.cache_write(cache, x.to(device), fmt=fmt)
    assert torch.equal(cache.cpu(), want)
    for out in DTYPES:
        back = ops.cache_read(cache, dim, fmt=fmt, dtype=out)
        assert back.dtype == out and back.shape == (n, dim)
        assert torch.equal(back.cpu(), R.cache_read(want, dim, fmt=fmt,
                                                    dtype=out))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("dim", [3, 64])
def test_slots_padding_and_repeats(device, fmt, index, dim):
    g = torch.Generator().manual_seed(dim)
    rows, n = 50, 300
    slots = torch.randint(-3, rows + 3, (n,), generator=g)
    x = torch.randn(n, dim, generator=g)
    start = torch.randint(0, 120, (rows, ops.record_bytes(dim)),
                          generator=g).to(torch.uint8)
    want = start.clone()
    for j in range(n):  # one after the other: the last one is kept
        s = int(slots[j])
        if 0 <= s < rows:
            R.cache_write(want[s:s + 1], x[j:j + 1], fmt=fmt)
    cache = start.to(device)
    ops.cache_write(cache, x.to(device), slots.to(device, index), fmt=fmt)
    assert torch.equal(cache.cpu(), want)
    back = ops.cache_read(cache, dim, slots.to(device, index), fmt=fmt).cpu()
    held = (slots >= 0) & (slots < rows)
    whole = R.cache_read(want, dim, fmt=fmt)
    assert torch.equal(back[held], whole[slots[held]])
    assert int(back[~held].abs().sum()) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_unique_writes_touch_only_their_slots(device):
    g = torch.Generator().manual_seed(1)
    slots = torch.randperm(40, generator=g)[:17]
    x = torch.randn(17, 12, generator=g)
    a = torch.full((40, ops.record_bytes(12)), 7, dtype=torch.uint8,
                   device=device)
    b = a.clone()
    ops.cache_write(a, x.to(device), slots.to(device), unique=True)
    ops.cache_write(b, x.to(device), slots.to(device))
    assert torch.equal(a, b)
    rest = torch.ones(40, dtype=torch.bool)
    rest[slots] = False
    assert bool((a.cpu()[rest] == 7).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_strided_operands(device, fmt):
    dim, n = 30, 21
    rec = ops.record_bytes(dim)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(n, dim, generator=g)
    want = ops.row_cache(n, dim)
    R.cache_write(want, x, fmt=fmt)
    x = x.to(device)
    wide = torch.zeros(n, 2 * dim + 1, device=device)
    wide[:, 3:3 + dim] = x
    sideways = x.t().contiguous().t()
    for values in (wide[:, 3:3 + dim], sideways, x[None].expand(2, n, dim)[1]):
        host = torch.full((n, rec + 12), 9, dtype=torch.uint8, device=device)
        cache = host[:, 8:8 + rec]
        ops.cache_write(cache, values, fmt=fmt)
        assert torch.equal(cache.cpu(), want)
        assert bool((host[:, :8] == 9).all()) and \
            bool((host[:, 8 + rec:] == 9).all())
        slots = torch.arange(2 * n, device=device)[::2] // 2
        assert torch.equal(
            ops.cache_read(cache, dim, slots, fmt=fmt).cpu(),
            R.cache_read(want, dim, fmt=fmt))


@pytest.mark.parametrize("device", DEVICES)
def test_empty(device):
    empty = ops.row_cache(0, 5, device)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    ops.cache_write(empty, torch.zeros(0, 5, device=device))
    ops.cache_write(empty, torch.zeros(0, 5, device=device), none)
    assert ops.cache_read(empty, 5).shape == (0, 5)
    assert ops.cache_read(empty, 5, none).shape == (0, 5)
    # a cache without records: every slot is padding
    some = torch.tensor([0, 3], device=device)
    ops.cache_write(empty, torch.ones(2, 5, device=device), some)
    assert int(ops.cache_read(empty, 5, some).abs().sum()) == 0
    # records that nothing was written to
    assert int(ops.cache_read(ops.row_cache(3, 5, device), 5,
                              fmt="fp8").abs().sum()) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.ones(4, 6, device=device)
    cache = ops.row_cache(4, 6, device)
    two = torch.tensor([0, 1], device=device)
    before = cache.clone()
    for bad in (lambda: ops.cache_write(cache, x, fmt="int4"),
                lambda: ops.cache_write(cache, x.double()),
                lambda: ops.cache_write(cache, x[0]),
                lambda: ops.cache_write(cache, x[:3]),
                lambda: ops.cache_write(cache, x[:, :1]),
                lambda: ops.cache_write(cache, x, two),
                lambda: ops.cache_write(cache, x[:2], two.float()),
                lambda: ops.cache_write(cache, x[:2], two[None]),
                lambda: ops.cache_write(cache.float(), x),
                lambda: ops.cache_write(cache[0], x),
                lambda: ops.cache_write(cache[:1].expand(4, 12), x),
                lambda: ops.cache_read(cache, 3),
                lambda: ops.cache_read(cache, 0),
                lambda: ops.cache_read(cache, 6, fmt="fp16"),
                lambda: ops.cache_read(cache, 6, dtype=torch.float64),
                lambda: ops.cache_read(cache, 6, two.float()),
                lambda: ops.row_cache(-1, 6), lambda: ops.row_cache(4, 0)):
        with pytest.raises(ValueError):
            bad()
    # records that are not 4-byte aligned
    loose = torch.zeros(4 * 13 + 1, dtype=torch.uint8, device=device)
    with pytest.raises(ValueError):
        ops.cache_write(loose[1:49].view(4, 12), x)
    with pytest.raises(ValueError):
        ops.cache_read(loose[:52].view(4, 13)[:, :12], 6)
    with pytest.raises(RuntimeError):
        ops.cache_write(cache, x.clone().requires_grad_())
    with torch.no_grad():
        ops.cache_write(before.clone(), x.clone().requires_grad_())
    assert torch.equal(cache, before)


@pytest.mark.gpu
def test_refuses_mixed_devices():
    with pytest.raises(ValueError):
        ops.cache_write(ops.row_cache(2, 4, "cuda"), torch.ones(2, 4))
    with pytest.raises(ValueError):
        ops.cache_read(ops.row_cache(2, 4, "cuda"), 4, torch.tensor([1]))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_records_beyond_32_bits(fmt):
    """Slots, bytes and elements past 2^31 and 2^32."""
    rows, dim = 9000000, 508  # 4.6e9 bytes
    cache = torch.empty(rows, ops.record_bytes(dim), dtype=torch.uint8,
                        device="cuda")
    g = torch.Generator().manual_seed(5)
    x = torch.randn(64, dim, generator=g)
    slots = torch.cat([torch.arange(rows - 40, rows),
                       torch.arange(0, 24) * 370000])
    ops.cache_write(cache, x.cuda(), slots.cuda(), fmt=fmt)
    want = ops.row_cache(64, dim)
    R.cache_write(want, x, fmt=fmt)
    assert torch.equal(cache[slots.cuda()].cpu(), want)
    back = ops.cache_read(cache, dim, slots.cuda(), fmt=fmt).cpu()
    assert torch.equal(back, R.cache_read(want, dim, fmt=fmt))


@pytest.mark.gpu
def test_side_stream_and_replayed_graph():
    dim, n = 48, 100
    cache = ops.row_cache(200, dim, "cuda")
    x = torch.randn(n, dim, device="cuda")
    slots = torch.randint(0, 200, (n,), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.cache_write(cache, x, slots, fmt="fp8")
        ops.cache_read(cache, dim, slots, fmt="fp8")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_write(cache, x, slots, fmt="fp8")
        out = ops.cache_read(cache, dim, slots, fmt="fp8")
    for k in range(4):
        x.copy_(torch.randn(n, dim, device="cuda"))
        slots.copy_(torch.randint(0, 200, (n,), device="cuda"))
        eager = cache.clone()
        graph.replay()
        torch.cuda.synchronize()
        ops.cache_write(eager, x, slots, fmt="fp8")
        assert torch.equal(cache, eager)
        assert torch.equal(out, ops.cache_read(eager, dim, slots, fmt="fp8"))


# -- the wire ------------------------------------------------------------

class PullPush(WorkerLogic):
    """Pulls its rows, keeps the answers, pushes given deltas."""

    def __init__(self, deltas):
        self.deltas = deltas
        self.seen = {}

    def on_recv(self, ids, client):
        client.pull(ids)

    def on_pull_recv(self, ids, values, client):
        for i, v in zip(ids.tolist(), values):
            self.seen[i] = v.clone()
        client.push(ids, self.deltas[ids])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wire,fmt", [("int8", "int8"), ("e4m3", "fp8")])
@pytest.mark.parametrize("feedback", ["fresh", "merged", "pipelined"])
def test_wire_carries_records(device, wire, fmt, feedback):
    """Rows of the other shard arrive as their records' values, own rows as
    they are; deltas likewise; bytes are those of the records."""
    world, num, dim = 2, 10, 7
    g = torch.Generator().manual_seed(4)
    deltas = torch.randn(num, dim, generator=g).to(device)

    def job(rank, transport):
        part = ModPartitioner(num, world)
        table = ShardedTable(part, rank, dim, device, init=(-1.0, 1.0))
        start = table.data.clone()
        logic = PullPush(deltas)
        eng = PSEngine(PSConfig(num_ids=num, dim=dim, wire_dtype=wire,
                                feedback=feedback), logic,
                       TableServerLogic(table, dump_on_close=False),
                       transport, part, device=device)
        eng.run([torch.arange(num, device=device)] if rank == 0 else [])
        return start, table.data.clone(), logic.seen, eng.metrics.bytes_sent

    def through(x):
        cache = ops.row_cache(x.shape[0], dim, device)
        ops.cache_write(cache, x.contiguous(), fmt=fmt)
        return ops.cache_read(cache, dim, fmt=fmt)

    (s0, t0, seen, sent), (s1, t1, _, answered) = run_loopback(world, job)
    assert sorted(seen) == list(range(num))
    got0 = torch.stack([seen[i] for i in range(0, num, 2)])
    got1 = torch.stack([seen[i] for i in range(1, num, 2)])
    assert torch.equal(got0, s0)
    assert torch.equal(got1, through(s1))
    assert torch.equal(t0, s0 + deltas[0::2])
    assert torch.equal(t1, s1 + through(deltas[1::2]))
    rec = ops.record_bytes(dim)
    assert sent == 5 * 8 + 5 * 8 + 5 * rec  # pull ids, push ids, deltas
    assert answered == 5 * rec


def test_config_refuses_unknown_wire():
    with pytest.raises(ValueError):
        PSConfig(wire_dtype="int4")
