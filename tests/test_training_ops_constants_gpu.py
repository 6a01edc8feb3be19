"""Calls of layer norm and the recurrence inside a vmap or beside forward-mode tangents, on tensors that take no part in
them: as ever.  (torch.func.grad and jvp wrap every new tensor, which has no address for a kernel then: refused.)"""
import pytest
import torch
import torch.autograd.forward_ad as fw

from conftest import pkg_module

pytestmark = pytest.mark.gpu


def test_constants_inside_transforms(cuda):
    ln, rec = pkg_module("layernorm"), pkg_module("recurrence")
    c = torch.randn(5, 3, 16, device=cuda)
    state = torch.randn(3, 16, device=cuda)
    x = torch.randn(4, device=cuda)
    for f in (lambda: ln.layer_norm(c), lambda: rec.gated_scan(c, c)[0], lambda: rec.linear_scan(c, c, state)[1],
              lambda: rec.gated_step(c[0], c[0], state.clone())):
        want = f().sum()
        run = lambda a: a * f().sum()
        assert torch.equal(torch.vmap(run)(x), x * want)
        with fw.dual_level():
            y = fw.unpack_dual(run(fw.make_dual(x, torch.ones_like(x))))
            assert torch.equal(y.tangent, want.expand(4))
        for transform in (lambda: torch.func.grad(lambda a: run(a).sum())(x), lambda: torch.func.jvp(run, (x,), (x,))):
            with pytest.raises(RuntimeError):
                transform()
