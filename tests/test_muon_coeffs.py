"""Coefficients that take singular values near zero further down."""
import pytest
import torch

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SHAPES = [(40, 60), (900, 128), (300, 900), (400, 520), (520, 800)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("steps,coeffs", [
    (60, (0.5, 0.0, 0.0)), (13, (0.5, 0.0, 0.0)), (8, (0.1, 0.2, 0.1)),
    (1, (0.0, 1.0, 0.0)), (4, (0.0, 3.0, -2.0)), (1, (2e-4, 0.5, 0.5)),
    (100, (-0.9, 0.1, 0.0))])
def test_refused(device, steps, coeffs):
    """Below 2^-12 they leave the bits that the kernels hold."""
    x = torch.ones(4, 6, device=device)
    with pytest.raises(ValueError, match="shrink"):
        ops.orthogonalize(x, steps=steps, coeffs=coeffs)
    with pytest.raises(ValueError, match="shrink"):
        ops.apply_muon(x, torch.zeros_like(x),
                       torch.arange(4, device=device), x.clone(), 0.1,
                       steps=steps, coeffs=coeffs)
    assert bool((x == 1).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("steps,coeffs", [
    (12, (0.5, 0.0, 0.0)), (3, (0.1, 0.2, 0.1)), (70, (0.9, -0.1, 0.0)),
    (70, (-0.9, 0.1, 0.0)), (100, (1.0, 0.0, 0.0)), (1, (0.0003, 0.5, 0.4))])
@pytest.mark.parametrize("m,n", SHAPES)
def test_taken(device, steps, coeffs, m, n):
    """No step multiplies one direction by more than a few times what it does
    to another (singular values of a random matrix are below 0.3), so that
    errors stay relative to the result: 2^-20 a step and at both ends, as two
    planes of 22 bits and f32 sums have it; the last coefficients, whose
    result lies in the square of the values, hold them to 2^-37 of P, which is
    3e-4 to 0.04."""
    a, b, c = coeffs
    g = torch.Generator().manual_seed(m)
    x = torch.randn(1, m, n, generator=g)
    want = x[0].double()
    want = want / (want.norm() + 1e-7)
    for _ in range(steps):
        if m <= n:
            s = want @ want.t()
            want = a * want + (b * s + c * s @ s) @ want
        else:
            s = want.t() @ want
            want = a * want + want @ (b * s + c * s @ s)
    got = ops.orthogonalize(x.to(device), steps=steps, coeffs=coeffs)[0]
    off = float((got.cpu().double() - want).norm() / want.norm())
    assert off <= (steps + 2) * 2.0 ** -20
