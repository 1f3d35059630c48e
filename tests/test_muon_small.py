"""Matrices whose norm is small beside eps.

X = U / (|U| + eps) is then small, and a step multiplies it by a: the result
is a^5 X but for terms of a (a^5 X)^2 relative to it.  Its error is relative
to itself: a step rounds X and the factor to 22 bits each (2^-22 off at most,
two halves of the last place of either included), leaves out a product of two
lows (2^-22) and adds sums of f32, a few 2^-24: 2^-20 in all at most, and as
much for X and for the result.  Planes keep an absolute 2^-37 of a matrix
whose norm is between 1/4 and 1: sqrt(m n) 2^-35 of it.
"""
import pytest
import torch

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SHAPES = [(12, 30), (900, 40), (500, 100), (100, 900), (300, 140), (400, 520),
          (150, 390)]
NORMS = [5e-12, 5e-14, 5e-16, 1e-25, 1e-36]


def exact(u, steps, eps):
    a, b, c = ops.MUON_COEFFS
    x = u.double()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        g = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
        q = b * g + c * g @ g
        x = a * x + (q @ x if x.shape[0] <= x.shape[1] else x @ q)
    return x


def limit(m, n, steps, dtype=torch.float32):
    floor = (m * n) ** 0.5 * 2.0 ** -35
    rounding = 0 if dtype is torch.float32 else torch.finfo(dtype).eps / 2
    return (steps + 2) * (2.0 ** -20 + floor) + rounding


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", SHAPES)
def test_small_beside_eps(device, dtype, m, n, norm):
    """The others of the batch are of ordinary size."""
    g = torch.Generator().manual_seed(m)
    x = torch.randn(3, m, n, generator=g)
    x[1] *= norm / float(x[1].norm())
    x = x.to(dtype)
    got = ops.orthogonalize(x.to(device)).cpu()
    want = exact(x[1], 5, 1e-7)
    off = float((got[1].double() - want).norm() / want.norm())
    assert off <= limit(m, n, 5, dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", [(900, 40), (100, 900), (400, 520)])
def test_small_in_many_steps(device, m, n):
    """Ten steps from 1e-13 of eps, in rounds of them on the thin routes: the
    values reach 2e-8."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, m, n, generator=g)
    x *= 1e-20 / float(x.norm())
    got = ops.orthogonalize(x.to(device), steps=10).cpu()
    want = exact(x[0], 10, 1e-7)
    off = float((got[0].double() - want).norm() / want.norm())
    assert off <= limit(m, n, 10)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", [(300, 20), (700, 100), (300, 140),
                                 (100, 700)])
def test_small_updates_of_a_table(device, m, n):
    g = torch.Generator().manual_seed(m + n)
    grads = torch.randn(m, n, generator=g)
    grads *= 5e-15 / float(grads.norm())
    table = torch.zeros(m, n, device=device)
    momentum = torch.zeros_like(table)
    ops.apply_muon(table, momentum, torch.arange(m, device=device),
                   grads.to(device), 0.5, mu=0.0, sorted_unique=True)
    want = -0.5 * max(1.0, m / n) ** 0.5 * exact(grads, 5, 1e-7)
    off = float((table.cpu().double() - want).norm() / want.norm())
    # and the rate's rounding, the product's with it
    assert off <= limit(m, n, 5) + 2 * 2.0 ** -24
