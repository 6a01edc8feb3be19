"""Single steps of the recurrence under torch's transforms of calls, on a B200: refused."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from conftest import pkg_module

pytestmark = pytest.mark.gpu


def test_single_steps_refuse(cuda):
    """The step writes its state in place and records nothing: it says so."""
    rec = pkg_module("recurrence")
    g, x = torch.randn(3, 16, device=cuda), torch.randn(3, 16, device=cuda)
    state = torch.randn(3, 16, device=cuda)
    keep = state.clone()
    for step in (rec.gated_step, rec.linear_step):
        with fw.dual_level():
            dual = fw.make_dual(x, torch.ones_like(x))
            for args in ((dual, x, state), (g, dual, state), (g, x, fw.make_dual(state, torch.ones_like(x)))):
                with pytest.raises(RuntimeError):
                    step(*args)
        with pytest.raises(RuntimeError):
            torch.jit.trace(lambda g, x: step(g, x, state), (g, x), check_trace=False)
        with pytest.raises(RuntimeError):
            torch.vmap(lambda g, x, s: step(g, x, s))(*(t[None] for t in (g, x, state)))
    assert torch.equal(state, keep)
    with fw.dual_level():                                  # nothing with a tangent among the arguments
        a = rec.gated_step(g, x, state)
    assert torch.equal(a, rec.gated_step(g, x, keep))
