"""Matrices of zeros under any eps that is accepted: zeros, and not NaN."""
import pytest
import torch

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# widths of the narrow, the thin and the wide routes, both orientations
SHAPES = [(12, 30), (900, 40), (500, 100), (100, 500), (300, 140), (140, 300)]
# where five steps take a singular value of one (0.696); off by half a place
# of bfloat16, 2^-8, at most
a, b, c = ops.MUON_COEFFS
ONE = 1.0
for _ in range(5):
    ONE *= a + b * ONE ** 2 + c * ONE ** 4
EPS = [1e-7, 1e-40, 1e-60, 2.2250738585072014e-308, 5e-324]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("m,n", SHAPES)
def test_zeros_give_zeros(device, dtype, m, n):
    x = torch.zeros(3, m, n, dtype=dtype, device=device)
    x[1, 0, 0] = 1
    for eps in EPS:
        got = ops.orthogonalize(x, eps=eps)
        assert bool((got[::2] == 0).all()), eps
        # 1 / (1 + 1e-7) moves as little as f32 does
        assert abs(float(got[1].float().norm()) / ONE - 1) <= 2 ** -8 + 1e-5


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_a_step_without_a_gradient_only_decays(device, m, n):
    table = torch.randn(2 * m, n, device=device)
    for eps in EPS:
        t, mo = table.clone(), torch.zeros_like(table)
        ops.apply_muon(t, mo, torch.arange(0, m, 3, device=device),
                       torch.zeros((m + 2) // 3, n, device=device), 0.5,
                       weight_decay=0.5, matrix_rows=m, eps=eps)
        # 1 - lr weight_decay = 3/4: one rounding a value
        assert torch.equal(t[:m], table[:m] * 0.75), eps
        assert torch.equal(t[m:], table[m:])
        assert int(mo.abs().sum()) == 0
