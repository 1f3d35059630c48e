"""Operators without a derivative refuse tensors that carry a tangent, which
would be lost without a word."""
import pytest
import torch
from torch.autograd import forward_ad

from flink_parameter_server_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_tangents_are_refused(device):
    x = torch.randn(6, 4, device=device)
    cache = ops.row_cache(6, 4, device)
    rows = torch.arange(6, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone(), torch.ones_like(x))
        for bad in (lambda: ops.orthogonalize(dual),
                    lambda: ops.orthogonalize(dual[None].mT),
                    lambda: ops.cache_write(cache, dual),
                    lambda: ops.apply_muon(x, torch.zeros_like(x), rows, dual,
                                           0.1),
                    lambda: ops.apply_muon(dual, torch.zeros_like(x), rows, x,
                                           0.1),
                    lambda: ops.apply_muon(x, dual, rows, x, 0.1)):
            with pytest.raises(RuntimeError, match="no gradient"):
                bad()
        assert int(cache.sum()) == 0
        # others are taken at a dual level as anywhere
        ops.orthogonalize(x)
        ops.cache_write(cache, x)
        ops.cache_read(cache, 4)
        ops.apply_muon(x.clone(), torch.zeros_like(x), rows, x, 0.1)
        ops.orthogonalize(forward_ad.unpack_dual(dual).primal)


@pytest.mark.parametrize("device", DEVICES)
def test_function_transforms_are_refused(device):
    x = torch.randn(6, 4, device=device)
    with pytest.raises(RuntimeError):
        torch.func.jvp(ops.orthogonalize, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: ops.orthogonalize(v).sum())(x)
