"""How far below a row's largest value fp8 records hold 2^-4 relative.

The largest value is more than 224 scales and codes have their full three bits
from 2^-6 scales up, so from 2^-6 / 224 = 1 / 14336 of the largest up.  Just
below, 7.5 * 2^-9 scales are off by 1 / 15.
"""
import pytest
import torch

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_relative_error_down_to_one_14336th(device):
    # the largest at the ends of what a scale takes, the others in all steps
    # from a third of the bound to three times it and up to the largest
    tops = torch.tensor([224.0, 224.00002, 225.0, 300.0, 447.9, 448.0,
                         448.00003, 460.0])
    small = torch.linspace(1 / 3, 3, 400) / 14336
    large = torch.logspace(-4, 0, 400).clamp(max=1.0)
    part = torch.cat([small, large])
    for power in (-118, -30, 0, 60, 119):
        x = torch.cat([tops[:, None], tops[:, None] * part], 1)
        x = x * 2.0 ** (power - 8)  # 224 is less than 2^8
        x[:, 1::2] *= -1
        cache = ops.row_cache(*x.shape, device)
        ops.cache_write(cache, x.to(device), fmt="fp8")
        back = ops.cache_read(cache, x.shape[1], fmt="fp8").cpu().double()
        x = x.double()
        size, top = x.abs(), x.abs().amax(1, keepdim=True)
        off = (back - x).abs()
        held = size * 14336 >= top
        assert bool((off <= size / 16)[held].all())
        # below, half of the smallest step: 2^-10 scales
        assert bool((off <= top / 224 * 2.0 ** -10)[~held].all())


@pytest.mark.parametrize("device", DEVICES)
def test_the_bound_is_where_it_ends(device):
    x = torch.tensor([[225.0, 7.5 * 2.0 ** -9]], device=device)
    cache = ops.row_cache(1, 2, device)
    ops.cache_write(cache, x, fmt="fp8")
    back = ops.cache_read(cache, 2, fmt="fp8")
    assert float(back[0, 1]) == 2.0 ** -6  # to the even neighbour: 1 / 15 off
