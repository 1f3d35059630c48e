"""Newton-Schulz orthogonalisation and the Muon apply (ops.orthogonalize,
ops.apply_muon) against the definition in 64 bits, their refusals, and the
server table that steps with them.

Tolerances.  A step f(X) = aX + bXX'X + cXX'XX'X moves a perturbation of X by
at most D = max |f'| over the singular values (its divided differences are
bounded by the derivative on [0, max s]); with the Muon coefficients and
s <= 1.3, D <= 3.4445.  Each step adds an error of at most delta |X|_F:
16 units of 2^-24 for the operands' rounding (two 22-bit planes in each of
three products, their dropped low products, or f32 itself, which is less) and
one for each of the K / 32 f32 additions of a sum over K.  To first order
    |error|_F <= delta * sum_k D^(steps - k) |X_k|_F,
which `bound` adds up with the exact X_k.  Values are kept down to 2^-37 of
the norm, which adds sqrt(m n) 2^-37 to each term.  A 16-bit result is rounded
once: half its eps relative to the result.
"""
import math

import numpy as np
import pytest
import torch

from flink_parameter_server_amd import (ModPartitioner, PSConfig, PSEngine,
                                        RangePartitioner, ShardedTable,
                                        TableServerLogic, WorkerLogic,
                                        load_shard, ops, save_shard)
from flink_parameter_server_amd.parallel.transport import run_loopback

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def chain(x, steps=5, coeffs=ops.MUON_COEFFS, eps=1e-7):
    """(result, bound) of one matrix in 64 bits."""
    a, b, c = coeffs
    x = x.double().cpu()
    x = x / (x.norm() + eps)
    m, n = x.shape
    if m > n:
        x = x.t()
    grid = torch.linspace(0, 1.3, 2000, dtype=torch.float64) ** 2
    D = float((a + 3 * b * grid + 5 * c * grid * grid).abs().max())
    delta = (16 + max(m, n) / 32) * U
    floor = math.sqrt(m * n) * 2.0 ** -37
    limit = 0.0
    for _ in range(steps):
        limit = D * (limit + delta * float(x.norm()) + floor)
        g = x @ x.t()
        x = a * x + (b * g + c * g @ g) @ x
    limit += delta * float(x.norm())
    return (x.t() if m > n else x), limit


def check(got, x, **kw):
    want, limit = chain(x, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    if got.dtype != torch.float32:
        limit += torch.finfo(got.dtype).eps / 2 * float(want.norm())
    off = float((got.double().cpu() - want).norm())
    assert off <= limit, (off, limit)


def matrices(kind, b, m, n, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, m, n, generator=g)
    if kind == "decay":  # a few strong directions
        r = min(m, n, 8)
        left = torch.randn(b, m, r, generator=g)
        left /= torch.arange(1, r + 1)
        x = torch.bmm(left, torch.randn(b, r, n, generator=g)) + 0.05 * x
    if kind == "steep":  # four directions a thousand times the others
        x = 1e-3 * x + torch.bmm(torch.randn(b, m, 4, generator=g),
                                 torch.randn(b, 4, n, generator=g))
    return x


SIZES = [(1, 1, 1), (1, 1, 50), (1, 50, 1), (4, 3, 5), (2, 16, 16),
         (3, 17, 33), (2, 64, 63), (1, 2000, 7), (1, 7, 2000), (1, 2500, 48),
         (1, 65, 65), (2, 100, 130), (2, 130, 100), (2, 200, 129),
         (1, 257, 300), (1, 4200, 130), (1, 130, 4200), (2, 128, 520),
         (2, 520, 128), (5, 128, 520)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["normal", "decay"])
@pytest.mark.parametrize("b,m,n", SIZES)
def test_orthogonalize(device, kind, b, m, n):
    x = matrices(kind, b, m, n, m + n)
    got = ops.orthogonalize(x.to(device))
    for k in range(b):
        check(got[k], x[k])


@pytest.mark.gpu
@pytest.mark.parametrize("b,m,n", [(1, 1024, 1024), (3, 300, 1001),
                                   (1, 700, 513), (1, 30000, 300),
                                   (1, 300, 30000), (1, 100000, 32),
                                   (2, 2048, 320), (1, 321, 11000),
                                   (1, 1500, 1400)])
def test_orthogonalize_large(b, m, n):
    x = matrices("decay", b, m, n, 1)
    got = ops.orthogonalize(x.cuda())
    for k in range(b):
        check(got[k], x[k])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("b,m,n", [
    (1, 130, 390), (1, 390, 130), (1, 224, 672), (1, 225, 675), (1, 673, 224),
    (1, 257, 800), (1, 320, 961), (1, 961, 320), (1, 256, 2048),
    (3, 400, 129), (2, 225, 1800), (4, 3300, 200), (8, 70, 1121),
    (9, 64, 66), (9, 65, 220)])
def test_where_the_routes_meet(b, m, n, dtype):
    x = matrices("decay", b, m, n, 15).to(dtype)
    got = ops.orthogonalize(x.cuda())
    for k in range(b):
        check(got[k], x[k])


@pytest.mark.gpu
def test_more_matrices_than_a_launch():
    """The last one, in a launch of its own, takes the others' route."""
    x = torch.randn(32769, 65, 200, device="cuda", dtype=torch.float16)
    got = ops.orthogonalize(x, steps=9)
    for k in (0, 20000, 32767, 32768):
        check(got[k], x[k].cpu(), steps=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [6, 7, 12, 13, 20, 100])
@pytest.mark.parametrize("m,n", [(24, 40), (2000, 40), (600, 128),
                                 (128, 600), (9000, 200), (150, 170)])
def test_many_steps(m, n, steps, dtype):
    """However often steps multiply what is small, the result stays near the
    one in 64 bits: at most eight times as far as the oracle's f32 steps are
    (which keep every value in f32 and round as often)."""
    x = matrices("normal", 1, m, n, 14).to(dtype)
    want = chain(x[0], steps=steps)[0]
    got = ops.orthogonalize(x.cuda(), steps=steps).cpu()
    f32 = ops.orthogonalize(x.float(), steps=steps)
    limit = 8 * float((f32[0].double() - want).norm())
    if dtype != torch.float32:
        limit += torch.finfo(dtype).eps / 2 * float(want.norm())
    off = float((got[0].double() - want).norm())
    assert off <= limit


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(6040, 32), (32, 6040), (4000, 60),
                                 (20000, 100), (100, 20000), (9000, 200),
                                 (700, 600), (600, 700)])
def test_no_element_stands_out(m, n):
    """An element's error is a sum of many roundings of its own; one that
    came of a value lost, or rounded in two ways, is hundreds of times the
    others (normal errors: 6 times their root mean square in 10^6)."""
    x = matrices("decay", 1, m, n, 13)
    off = (ops.orthogonalize(x.cuda())[0].double().cpu() - chain(x[0])[0])
    assert float(off.abs().max()) <= 32 * float(off.square().mean().sqrt())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n", [(20, 90), (90, 20), (150, 170), (170, 150)])
def test_16_bit_types(device, dtype, m, n):
    x = matrices("normal", 2, m, n, 3).to(dtype)
    got = ops.orthogonalize(x.to(device))
    for k in range(2):
        check(got[k], x[k])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["normal", "decay", "steep"])
@pytest.mark.parametrize("steps,coeffs", [(1, ops.MUON_COEFFS),
                                          (2, ops.MUON_COEFFS),
                                          (5, ops.MUON_COEFFS),
                                          (8, ops.MUON_COEFFS),
                                          (11, ops.MUON_COEFFS),
                                          (3, (1.5, -0.5, 0.0)),
                                          (9, (1.875, -1.25, 0.375))])
@pytest.mark.parametrize("m,n", [(140, 300), (300, 140), (130, 2100),
                                 (520, 790)])
def test_long_bfloat16_matrices(device, kind, steps, coeffs, m, n):
    """Some steps in a row may be taken on the Gram matrix where that stays
    below bfloat16's rounding, also where a few singular values are a thousand
    times the others: the error of the result is at most a tenth more than
    that of the exact result's rounding."""
    x = matrices(kind, 2, m, n, 12).bfloat16()
    got = ops.orthogonalize(x.to(device), steps=steps, coeffs=coeffs).cpu()
    for k in range(2):
        want, _ = chain(x[k], steps=steps, coeffs=coeffs)
        rounding = float((want.bfloat16().double() - want).norm())
        off = float((got[k].double() - want).norm())
        assert off <= 1.1 * rounding


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", [(24, 40), (90, 140)])
@pytest.mark.parametrize("steps,coeffs", [(1, ops.MUON_COEFFS),
                                          (2, ops.MUON_COEFFS),
                                          (3, (1.5, -0.5, 0.0)),
                                          (6, (2.0, -1.5, 0.5)),
                                          (12, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(device, steps, coeffs, m, n):
    x = matrices("normal", 1, m, n, 4)
    got = ops.orthogonalize(x.to(device), steps=steps, coeffs=coeffs)
    check(got[0], x[0], steps=steps, coeffs=coeffs)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", [(12, 30), (100, 140)])
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-9, 1e-7, 1e9, 1e30,
                                   1e37])
def test_magnitudes(device, scale, m, n):
    x = (matrices("normal", 1, m, n, 5).clamp(-3, 3) * scale)
    got = ops.orthogonalize(x.to(device))
    check(got[0], x[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", [(12, 30), (100, 140), (140, 100)])
def test_zeros_and_values_that_are_not_finite(device, m, n):
    x = matrices("normal", 5, m, n, 6)
    x[1] = 0
    x[2, m // 2, n // 2] = float("nan")
    x[3, 0, n - 1] = float("inf")
    got = ops.orthogonalize(x.to(device)).cpu()
    for k in (0, 4):  # the neighbours do not notice
        check(got[k], x[k])
    assert int(got[1].abs().sum()) == 0 and not bool(torch.isnan(got[1]).any())
    assert bool(torch.isnan(got[2]).all()) and bool(torch.isnan(got[3]).all())


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_and_strides(device):
    x = matrices("normal", 6, 20, 70, 7).to(device)
    want = ops.orthogonalize(x)
    assert torch.equal(ops.orthogonalize(x.view(2, 3, 20, 70)).view(6, 20, 70),
                       want)
    assert torch.equal(ops.orthogonalize(x[3]), want[3])
    sideways = x.mT.contiguous().mT
    kept = sideways.clone()
    assert torch.equal(ops.orthogonalize(sideways), want)
    assert torch.equal(sideways, kept)
    assert torch.equal(ops.orthogonalize(x[::2]), want[::2])
    for shape in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 5)):
        assert ops.orthogonalize(torch.zeros(shape, device=device)).shape \
            == shape


@pytest.mark.gpu
@pytest.mark.parametrize("b,m,n", [(3, 40, 60), (2, 3000, 40), (2, 200, 150)])
def test_results_do_not_depend_on_neighbours_or_runs(b, m, n):
    x = matrices("decay", b, m, n, 8).cuda()
    one = ops.orthogonalize(x)
    assert torch.equal(ops.orthogonalize(x), one)


@pytest.mark.gpu
def test_many_small_matrices():
    x = torch.randn(70000, 2, 3, device="cuda")
    got = ops.orthogonalize(x)
    for k in (0, 32767, 32768, 65535, 65536, 69999):
        check(got[k], x[k].cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_orthogonalize_refusals(device):
    x = torch.ones(3, 4, device=device)
    for bad in (lambda: ops.orthogonalize(x.double()),
                lambda: ops.orthogonalize(x[0]),
                lambda: ops.orthogonalize(x.long()),
                lambda: ops.orthogonalize(x, steps=0),
                lambda: ops.orthogonalize(x, steps=101),
                lambda: ops.orthogonalize(x, eps=0.0),
                lambda: ops.orthogonalize(x, eps=float("nan")),
                lambda: ops.orthogonalize(x, coeffs=(1.0, 2.0)),
                lambda: ops.orthogonalize(x, coeffs=(1.0, float("inf"), 0)),
                lambda: ops.orthogonalize(x, coeffs=(1.0, float("nan"), 0)),
                lambda: ops.orthogonalize(x, coeffs=(2.0, 0.0, 0.0)),
                lambda: ops.orthogonalize(x, coeffs=(16.0, -20.0, 0.0),
                                          steps=1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.orthogonalize(x.requires_grad_())
    with torch.no_grad():
        ops.orthogonalize(x)


# -- the apply -------------------------------------------------------------

def muon_by_hand(table, momentum, rows, grads, m, lr, mu, nesterov, wd):
    """(table, momentum, per-matrix (bound on the step's error, |W|_F)) in
    64 bits."""
    W, M = table.double().clone(), momentum.double().clone()
    n = W.shape[1]
    g = torch.zeros_like(W)
    inside = (rows >= 0) & (rows < W.shape[0])
    g.index_add_(0, rows[inside], grads[inside].double())
    limits = []
    for k in range(W.shape[0] // m):
        at = slice(k * m, (k + 1) * m)
        if not bool(((rows >= k * m) & (rows < (k + 1) * m)).any()):
            limits.append(None)
            continue
        M[at] = mu * M[at] + g[at]
        u = g[at] + mu * M[at] if nesterov else M[at]
        o, limit = chain(u)
        rate = lr * max(1.0, m / n) ** 0.5
        # U itself: a few f32 roundings, moved by the chain like X_0's
        limit += 8 * U * 3.4445 ** 5
        W[at] = (1 - lr * wd) * W[at] - rate * o
        limits.append(rate * limit + 8 * U * (
            float(table[at].double().norm()) + rate * float(o.norm())))
    return W, M, limits


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("matrices_,m,n,push", [
    (1, 40, 16, "all"), (1, 300, 8, "some"), (3, 20, 50, "repeats"),
    (4, 100, 120, "repeats"), (2, 150, 70, "all"), (5, 64, 64, "some"),
    (3, 1, 9, "all"), (1, 1, 1, "repeats"), (2, 70, 1, "some"),
    (2, 700, 200, "repeats"), (1, 200, 700, "some")])
def test_apply_muon(device, nesterov, matrices_, m, n, push):
    g = torch.Generator().manual_seed(m + n)
    R = matrices_ * m
    table = torch.randn(R, n, generator=g)
    momentum = torch.randn(R, n, generator=g) * 0.1
    if push == "all":
        rows = torch.arange(R)
    elif push == "some":
        rows = torch.randperm(R, generator=g)[:max(1, R // 3)].sort().values
    else:
        # matrix 1 is left alone, and some rows lie outside the table
        rows = torch.randint(-2, R + 2, (2 * R,), generator=g)
        if matrices_ > 1:
            rows[(rows >= m) & (rows < 2 * m)] = 0
    grads = torch.randn(rows.numel(), n, generator=g)
    W, M, limits = muon_by_hand(table, momentum, rows, grads, m, 0.05, 0.9,
                                nesterov, 0.1)
    t, mo = table.to(device), momentum.to(device)
    ops.apply_muon(t, mo, rows.to(device), grads.to(device), 0.05, mu=0.9,
                   nesterov=nesterov, weight_decay=0.1, matrix_rows=m,
                   sorted_unique=push != "repeats")
    t, mo = t.cpu(), mo.cpu()
    # a product, mu's own rounding, and the sum of up to d gradients
    d = int(torch.bincount(rows.clamp(min=0)).max())
    size = momentum.abs().max() + d * grads.abs().max()
    assert float((mo.double() - M).abs().max()) <= (3 + d) * U * float(size)
    for k, limit in enumerate(limits):
        at = slice(k * m, (k + 1) * m)
        if limit is None:
            assert torch.equal(t[at], table[at])
            assert torch.equal(mo[at], momentum[at])
        else:
            assert float((t[at].double() - W[at]).norm()) <= limit


@pytest.mark.parametrize("device", DEVICES)
def test_apply_muon_orders_and_index_types(device):
    g = torch.Generator().manual_seed(9)
    R, n = 60, 12
    table = torch.randn(R, n, generator=g).to(device)
    rows = torch.randint(0, R, (200,), generator=g).to(device)
    grads = torch.randn(200, n, generator=g).to(device)

    def step(rows, grads, **kw):
        t, m = table.clone(), torch.zeros_like(table)
        ops.apply_muon(t, m, rows, grads, 0.1, matrix_rows=20, **kw)
        return t, m

    one = step(rows, grads)
    two = step(rows.int(), grads)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    order = torch.sort(rows, stable=True).indices
    three = step(rows[order], grads[order])
    assert torch.equal(one[0], three[0]) and torch.equal(one[1], three[1])
    wide = torch.zeros(200, 2 * n, device=device)
    wide[:, ::2] = grads
    twice = torch.zeros(400, dtype=torch.int64, device=device)
    twice[::2] = rows
    four = step(twice[::2], wide[:, ::2])
    assert torch.equal(one[0], four[0]) and torch.equal(one[1], four[1])
    # none of the rows is in the table: nothing changes
    five = step(rows + R, grads)
    assert torch.equal(five[0], table) and int(five[1].abs().sum()) == 0
    six = step(rows[:0], grads[:0])
    assert torch.equal(six[0], table)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("matrices_,m,pushed,skew", [
    (1, 1000, 5000, 0.0), (3, 700, 16384, 0.6), (2, 300, 16385, 0.3),
    (2, 256, 513, 0.0), (2, 257, 3, 0.0), (1, 5, 16384, 0.0),
    (1024, 3, 700, 0.5), (1025, 3, 700, 0.5)])
def test_unsorted_pushes_sum_in_their_order(device, matrices_, m, pushed,
                                            skew):
    """M is mu M + g to the bit, with g summed in f32 in the push's order;
    pushes and tables on both sides of where they are sorted first."""
    g = torch.Generator().manual_seed(pushed + m)
    R, n, mu = matrices_ * m, 5, 0.5
    rows = torch.randint(-3, R + 3, (pushed,), generator=g)
    rows[torch.rand(pushed, generator=g) < skew] = R - 1
    grads = torch.randn(pushed, n, generator=g)
    mo = torch.randn(R, n, generator=g)
    total = np.zeros((R, n), dtype=np.float32)
    inside = (rows >= 0) & (rows < R)
    np.add.at(total, rows[inside].numpy(), grads[inside].numpy())
    named = torch.zeros(matrices_, dtype=torch.bool)
    named[rows[inside] // m] = True
    want = torch.where(named.repeat_interleave(m)[:, None],
                       mu * mo + torch.from_numpy(total), mo)
    t, v = torch.zeros(R, n, device=device), mo.to(device)
    ops.apply_muon(t, v, rows.to(device), grads.to(device), 0.1, mu=mu,
                   matrix_rows=m)
    assert torch.equal(v.cpu(), want)  # a product by 1/2 is exact
    assert torch.equal(t.cpu().view(matrices_, -1).any(1), named)


@pytest.mark.gpu
def test_more_matrices_than_a_grid():
    """1,100,000 matrices of one value: each is its own sign, five steps on."""
    R = 1100000
    u, w = torch.randn(R, 1), torch.randn(R, 1)
    t, v = w.cuda(), torch.zeros(R, 1, device="cuda")
    ops.apply_muon(t, v, torch.arange(R).cuda(), u.cuda(), 0.1, mu=0.0,
                   matrix_rows=1, sorted_unique=True)
    x = u.double() / (u.double().abs() + 1e-7)
    a, b, c = ops.MUON_COEFFS
    for _ in range(5):
        x = x * (a + b * x ** 2 + c * x ** 4)
    # P and U in two planes each (2^-22), their lows' product left out (2^-22),
    # f32 sums; then the weights' own roundings
    limit = 0.1 * 8 * 2.0 ** -22 * x.abs() + 2 * U * (w.abs() + 0.2).double()
    assert bool(((t.cpu().double() - (w.double() - 0.1 * x)).abs()
                 <= limit).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(300, 20), (700, 100)])
def test_apply_muon_many_steps(m, n):
    """The step's rounds end in the table, from the momentum's own pass."""
    g = torch.randn(m, n)
    table, mo = torch.randn(m, n), torch.randn(m, n)
    rows = torch.arange(m)
    t, v = table.cuda(), mo.cuda()
    ops.apply_muon(t, v, rows.cuda(), g.cuda(), 0.1, steps=9,
                   sorted_unique=True)
    M = 0.95 * mo.double() + g.double()
    step = ops.orthogonalize((g.double() + 0.95 * M).float(), steps=9)
    want = table.double() - 0.1 * math.sqrt(m / n) * step.double()
    # two f32 chains of nine steps, each off by at most `chain`'s bound
    limit = 2 * 0.1 * math.sqrt(m / n) * chain(g + 0.95 * M, steps=9)[1]
    off = float((t.cpu().double() - want).norm())
    assert off <= limit
    # near enough to say that no step is missing: one changes values by a
    # fifth of their size and more
    assert off <= 1e-3 * float((want - table.double()).norm())


@pytest.mark.gpu
def test_rows_that_are_not_sorted_as_promised_stay_inside():
    """A broken promise gives wrong sums, not a fault."""
    table = torch.randn(600, 8, device="cuda")
    mo = torch.zeros_like(table)
    rows = torch.randint(-5, 700, (900,), device="cuda")
    ops.apply_muon(table, mo, rows, torch.randn(900, 8, device="cuda"), 0.1,
                   matrix_rows=300, sorted_unique=True)
    assert bool(torch.isfinite(table).all())


@pytest.mark.parametrize("device", DEVICES)
def test_apply_muon_with_a_bad_gradient(device):
    """It takes its own matrix and no other."""
    table = torch.randn(40, 6, device=device)
    mo = torch.zeros_like(table)
    grads = torch.randn(40, 6, device=device)
    grads[3, 2] = float("nan")
    before = table.clone()
    ops.apply_muon(table, mo, torch.arange(40, device=device), grads, 0.1,
                   matrix_rows=10, sorted_unique=True)
    assert bool(torch.isnan(table[:10]).all())
    assert bool(torch.isfinite(table[10:]).all())
    assert not bool((table[10:] == before[10:]).all(1).any())


@pytest.mark.parametrize("device", DEVICES)
def test_apply_muon_refusals(device):
    t = torch.ones(6, 4, device=device)
    m = torch.zeros_like(t)
    r = torch.tensor([0, 1], device=device)
    g = torch.ones(2, 4, device=device)
    for bad in (lambda: ops.apply_muon(t, m, r, g, 0.1, matrix_rows=4),
                lambda: ops.apply_muon(t, m, r, g, 0.1, matrix_rows=0),
                lambda: ops.apply_muon(t, m[:3], r, g, 0.1),
                lambda: ops.apply_muon(t.double(), m, r, g, 0.1),
                lambda: ops.apply_muon(t, m.half(), r, g, 0.1),
                lambda: ops.apply_muon(t, t, r, g, 0.1),
                lambda: ops.apply_muon(t, m, r.float(), g, 0.1),
                lambda: ops.apply_muon(t, m, r[None], g, 0.1),
                lambda: ops.apply_muon(t, m, r, g[:, :3], 0.1),
                lambda: ops.apply_muon(t, m, r, g[:1], 0.1),
                lambda: ops.apply_muon(t, m, r, g.double(), 0.1),
                lambda: ops.apply_muon(t, m, r, g, 0.1, steps=0),
                lambda: ops.apply_muon(t.t(), m.t(), r, g, 0.1)):
        with pytest.raises(ValueError):
            bad()
    assert bool((t == 1).all()) and int(m.abs().sum()) == 0


@pytest.mark.gpu
def test_refuses_mixed_devices():
    t = torch.ones(6, 4, device="cuda")
    with pytest.raises(ValueError):
        ops.apply_muon(t, torch.zeros(6, 4), torch.tensor([0]),
                       torch.ones(1, 4), 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(96, 40), (160, 130)])
def test_side_stream_and_replayed_graphs(m, n):
    """Two captured graphs that share the pool, replayed in turn with eager
    work between, against eager results."""
    x = torch.randn(2, m, n, device="cuda")
    table, mo = torch.randn(m, n, device="cuda"), torch.zeros(m, n,
                                                              device="cuda")
    rows = torch.arange(m, device="cuda")
    grads = torch.randn(m, n, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = ops.orthogonalize(x)
        ops.apply_muon(table, mo, rows, grads, 0.1, sorted_unique=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, ops.orthogonalize(x))
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        out = ops.orthogonalize(x)
    with torch.cuda.graph(two, pool=one.pool()):
        ops.apply_muon(table, mo, rows, grads, 0.1, sorted_unique=True)
    for k in range(4):
        x.copy_(torch.randn(2, m, n, device="cuda"))
        grads.copy_(torch.randn(m, n, device="cuda"))
        t, v = table.clone(), mo.clone()
        one.replay()
        torch.cuda.synchronize()
        got = out.clone()
        two.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.orthogonalize(x))
        ops.apply_muon(t, v, rows, grads, 0.1, sorted_unique=True)
        assert torch.equal(table, t) and torch.equal(mo, v)


@pytest.mark.gpu
@pytest.mark.parametrize("matrices_,m,pushed", [(1, 300, 500), (3, 300, 16384),
                                                (1100, 2, 700)])
def test_unsorted_pushes_in_a_graph(matrices_, m, pushed):
    R, n = matrices_ * m, 6
    table, mo = (torch.randn(R, n, device="cuda") for _ in range(2))
    rows = torch.randint(-2, R + 2, (pushed,), device="cuda")
    grads = torch.randn(pushed, n, device="cuda")
    ops.apply_muon(table, mo, rows, grads, 0.1, matrix_rows=m)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.apply_muon(table, mo, rows, grads, 0.1, matrix_rows=m)
    for k in range(4):
        rows.copy_(torch.randint(-2, R + 2, (pushed,), device="cuda"))
        grads.copy_(torch.randn(pushed, n, device="cuda"))
        t, v = table.clone(), mo.clone()
        graph.replay()
        torch.cuda.synchronize()
        ops.apply_muon(t, v, rows, grads, 0.1, matrix_rows=m)
        assert torch.equal(table, t) and torch.equal(mo, v)


@pytest.mark.gpu
def test_a_push_that_needs_a_sort_is_not_captured():
    table, mo = torch.ones(300, 6, device="cuda"), torch.zeros(
        300, 6, device="cuda")
    rows = torch.randint(0, 300, (16385,), device="cuda")
    grads = torch.randn(16385, 6, device="cuda")
    one = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one += 1  # the graph has a node
        with pytest.raises(RuntimeError, match="captured"):
            ops.apply_muon(table, mo, rows, grads, 0.1)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((one == 1).all()) and bool((table == 1).all())
    ops.apply_muon(table, mo, rows, grads, 0.1)  # not captured: it steps
    assert not bool((table == 1).any())


# -- the server ------------------------------------------------------------

class Regress(WorkerLogic):
    """Pulls whole matrices, pushes the gradients of |W x - y|^2 / 2."""

    def __init__(self, ids, x, y):
        self.ids, self.x, self.y = ids, x, y
        self.pulled = []

    def on_recv(self, data, client):
        client.pull(self.ids, unique=True)

    def on_pull_recv(self, ids, values, client):
        order = torch.argsort(ids)
        w = values[order]
        self.pulled.append(w.clone())
        client.push(self.ids, (w @ self.x - self.y) @ self.x.t())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wire", ["f32", "int8", "e4m3"])
def test_weights_train_over_the_8_bit_wire(device, wire):
    """Two shards of two matrices each; one worker's pushes step them.  The
    engine's tables equal the same calls made by hand: rows answered through
    the wire, gradients pushed through it, one Muon step a push and shard."""
    world, count, m, n = 2, 4, 24, 10
    num, half = count * m, count * m // 2
    g = torch.Generator().manual_seed(11)
    x = torch.randn(n, 30, generator=g).to(device)
    y = torch.randn(num, 30, generator=g).to(device)
    ids = torch.arange(num, device=device)

    def job(rank, transport):
        part = RangePartitioner(num, world)
        table = ShardedTable(part, rank, n, device, init=(-0.1, 0.1),
                             optimizer="muon", lr=0.05, weight_decay=0.01,
                             matrix_rows=m)
        start = table.data.clone()
        logic = Regress(ids, x, y)
        eng = PSEngine(PSConfig(num_ids=num, dim=n, wire_dtype=wire,
                                partitioner="range"), logic,
                       TableServerLogic(table, dump_on_close=False,
                                        pushes_unique=True),
                       transport, part, device=device)
        eng.run([0, 0, 0] if rank == 0 else [])
        return start, table.data, table.accum, logic.pulled

    def through(v):
        if wire == "f32":
            return v
        cache = ops.row_cache(v.shape[0], n, device)
        fmt = {"int8": "int8", "e4m3": "fp8"}[wire]
        ops.cache_write(cache, v.contiguous(), fmt=fmt)
        return ops.cache_read(cache, n, fmt=fmt)

    (s0, t0, m0, pulled), (s1, t1, m1, _) = run_loopback(world, job)
    assert len(pulled) == 3
    W = torch.cat([s0, s1])
    M = torch.zeros_like(W)
    rows = torch.arange(half, device=device)
    pushes = [(w @ x - y) @ x.t() for w in pulled]
    for grad in pushes:
        for at, gr in ((slice(0, half), grad[:half]),
                       (slice(half, num), through(grad[half:]))):
            ops.apply_muon(W[at], M[at], rows, gr.contiguous(), 0.05,
                           weight_decay=0.01, matrix_rows=m,
                           sorted_unique=True)
    assert torch.equal(torch.cat([t0, t1]), W)
    assert torch.equal(torch.cat([m0, m1]), M)
    assert torch.equal(pulled[0], torch.cat([s0, through(s1)]))


def test_table_refuses_split_matrices():
    def table(part, shard=0, **kw):
        return ShardedTable(part, shard, 4, "cpu", optimizer="muon", lr=0.1,
                            **kw)
    assert table(ModPartitioner(12, 1)).matrix_rows == 12
    assert table(ModPartitioner(12, 1), matrix_rows=6).matrix_rows == 6
    assert table(RangePartitioner(24, 2), 1, matrix_rows=6).rows == 12
    assert table(ModPartitioner(12, 1), 1, matrix_rows=6).rows == 0
    for bad in (lambda: table(ModPartitioner(12, 1), matrix_rows=5),
                lambda: table(ModPartitioner(12, 1), matrix_rows=0),
                lambda: table(ModPartitioner(24, 2), matrix_rows=6),
                lambda: table(RangePartitioner(24, 2)),
                lambda: table(RangePartitioner(18, 2), matrix_rows=6),
                lambda: ShardedTable(ModPartitioner(4, 1), 0, 4, "cpu",
                                     optimizer="lion")):
        with pytest.raises(ValueError):
            bad()


def test_momentum_is_checkpointed(tmp_path):
    part = ModPartitioner(12, 1)
    one = ShardedTable(part, 0, 4, "cpu", init=(-1.0, 1.0), optimizer="muon",
                       lr=0.1, matrix_rows=6)
    ids = torch.arange(12)
    one.apply(ids, torch.randn(12, 4), unique=True)
    save_shard(str(tmp_path), one)
    two = ShardedTable(part, 0, 4, "cpu", optimizer="muon", lr=0.1,
                       matrix_rows=6)
    load_shard(str(tmp_path), two)
    g = torch.randn(12, 4)
    one.apply(ids, g)
    two.apply(ids, g)
    assert torch.equal(one.data, two.data)
    assert torch.equal(one.accum, two.accum)
