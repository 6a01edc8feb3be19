"""optim.AdamW's bookkeeping of groups and tensors, without a GPU: the check for CUDA parameters is replaced, and
nothing here launches a kernel."""
import pytest
import torch

from conftest import pkg_module


@pytest.fixture()
def optim(monkeypatch):
    mod = pkg_module("optim")
    monkeypatch.setattr(mod._lib, "require_cuda_tensor", lambda t, *a, **k: t)
    return mod


def param(n, grad=False):
    p = torch.zeros(n, requires_grad=True)
    if grad:
        p.grad = torch.ones(n)
    return p


def test_a_group_whose_state_cannot_be_made_is_not_kept(optim, monkeypatch):
    a, b = param(300), param(500)
    opt = optim.AdamW([a])
    state = dict(opt.state)

    def full(*args, **kw):
        raise torch.cuda.OutOfMemoryError("no room")

    with monkeypatch.context() as m:
        m.setattr(optim.torch, "zeros", full)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            opt.add_param_group({"params": [b]})
    assert len(opt.param_groups) == len(opt._buckets) == 1 and dict(opt.state) == state
    opt.add_param_group({"params": [b]})                   # there is room again
    assert len(opt.param_groups) == len(opt._buckets) == 2 and b in opt.state


def test_groups_changed_behind_the_optimiser_are_refused(optim):
    """Buckets are found by their group's place: a group taken out, or a tensor put into or out of one by hand, would
    update tensors with another group's numbers, or pass them by without a word."""
    def fresh():
        return optim.AdamW([{"params": [param(3), param(4)], "lr": 1e-2}, {"params": [param(5)]}], lr=1e-3)

    opt = fresh()
    opt.step()                                             # no gradients: nothing to do
    for change in (lambda o: o.param_groups.pop(0), lambda o: o.param_groups.append({**o.param_groups[0], "params": []}),
                   lambda o: o.param_groups.reverse(), lambda o: o.param_groups[1]["params"].append(param(6)),
                   lambda o: o.param_groups[0]["params"].pop(),
                   lambda o: o.param_groups[0]["params"].__setitem__(0, param(3))):
        opt = fresh()
        change(opt)
        with pytest.raises(RuntimeError):
            opt.step()
