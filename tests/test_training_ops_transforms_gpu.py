"""Layer norm and the recurrence under torch's transforms of calls, on a B200: forward-mode derivatives, traces
and vmap are refused or recorded, never passed by (an operator that fills its output behind torch's back
would have a zero tangent, and a trace of uninitialised memory)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from conftest import pkg_module

pytestmark = pytest.mark.gpu


def operators():
    ln, rec = pkg_module("layernorm"), pkg_module("recurrence")
    return {"layer_norm": lambda x: ln.layer_norm(x), "gated_scan": lambda x: rec.gated_scan(x, x)[0],
            "linear_scan": lambda x: rec.linear_scan(x, x)[1]}


NAMES = ["layer_norm", "gated_scan", "linear_scan"]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(cuda, name, grad):
    f = operators()[name]
    x = torch.randn(5, 3, 16, device=cuda)
    with torch.set_grad_enabled(grad), fw.dual_level():
        plain = f(x)                                       # no tangent: as ever
        assert torch.equal(plain, f(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(fw.make_dual(x, torch.randn_like(x)))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, (x,), (torch.randn_like(x),))


@pytest.mark.parametrize("name", NAMES)
def test_vmap_and_func_grad_are_refused(cuda, name):
    f = operators()[name]
    x = torch.randn(2, 5, 3, 16, device=cuda)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.vmap(f)(x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.grad(lambda x: f(x).sum())(x[0])


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.filterwarnings("ignore")
def test_a_trace_holds_the_operator(cuda, name, grad):
    f = operators()[name]
    x, other = torch.randn(5, 3, 16, device=cuda), torch.randn(5, 3, 16, device=cuda)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(f, (x,), check_trace=False)
        assert torch.equal(traced(other), f(other))
