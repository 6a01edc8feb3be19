"""layernorm.LayerNorm and layer_norm under torch.autocast on a B200: as torch's module there, computed and
returned in fp32, whatever the input's and the weights' types."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("xdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_as_torchs_module(cuda, kind, xdtype, wdtype):
    """Types as torch's, values as this module's own on fp32 copies (whose tests compare them with fp64)."""
    ln = pkg_module("layernorm")
    torch.manual_seed(0)
    mine = ln.LayerNorm(96, device=cuda, dtype=wdtype)
    with torch.no_grad():
        mine.weight.normal_()
        mine.bias.normal_()
    ref = torch.nn.LayerNorm(96, device=cuda, dtype=wdtype)
    ref.load_state_dict(mine.state_dict())
    x = torch.randn(7, 96, device=cuda).to(xdtype).requires_grad_()
    with torch.autocast("cuda", dtype=kind):
        y, z = mine(x), ref(x)
        direct = ln.layer_norm(x, mine.weight, mine.bias, mine.eps)
    assert y.dtype == z.dtype == torch.float32 and torch.equal(direct, y)
    plain = ln.layer_norm(x.float(), mine.weight.float(), mine.bias.float(), mine.eps)
    assert torch.equal(y, plain)
    dy = torch.randn_like(y)
    leaves = (x, mine.weight, mine.bias)
    for a, b, leaf in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(plain, leaves, dy), leaves):
        assert a.dtype == leaf.dtype and torch.equal(a, b)
    with torch.autocast("cuda", dtype=kind, enabled=False):
        if wdtype in (torch.float32, xdtype):
            assert mine(x).dtype == xdtype
