"""layernorm.layer_norm of constant 16-bit rows of more columns than a thread's fp32 chain adds up exactly, on a B200."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [131_073, 300_000, 2_000_001, 5_000_000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_constant_rows_give_the_bias(cuda, dim, dtype):
    """256 values of 11 bits add up exactly in fp32, their sums in fp64: the mean is the value, in every width."""
    ln = pkg_module("layernorm")
    g = torch.Generator(device=cuda).manual_seed(dim)
    x = (10 ** (2 + 2.75 * torch.rand(12, 1, device=cuda, generator=g))).to(dtype).expand(12, dim).contiguous()
    b = torch.randn(dim, device=cuda, generator=g)
    assert torch.equal(ln.layer_norm(x, None, b), b.to(dtype).expand(12, dim))
    assert bool((ln.layer_norm(x) == 0).all())
