"""Rows of layernorm.layer_norm whose squares pass fp32's range: finite, as torch's (whose 1 / deviation is zero then)."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [33, 184, 512, 4096, 9001, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_squares_past_the_range(cuda, dim, dtype):
    ln = pkg_module("layernorm")
    x = (torch.randn(9, dim, device=cuda) * 1e20).to(dtype).requires_grad_()
    w = torch.randn(dim, device=cuda, requires_grad=True)
    b = torch.randn(dim, device=cuda)
    y = ln.layer_norm(x, w, b)
    assert torch.equal(y, b.to(dtype).expand(9, dim))
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert bool((dx == 0).all()) and bool((dw == 0).all())
