"""optim.AdamW's flat state behind the tensors' ends, on a B200: zero, whatever the gradients hold."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu


def tails(opt, n):
    for name, flat in opt.state_buffers()[0].items():
        if name in ("exp_avg", "exp_avg_sq", "master"):
            yield name, flat[n:].float()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_tails_stay_zero_when_the_clip_is_nan(cuda, bits, dtype, value):
    """One gradient that is not finite makes the norm, and with it the clip's factor, NaN or zero: every element of
    the tensors is torch's own (NaN, or zero times infinity in one place), what lies behind them is zero."""
    optim = pkg_module("optim")
    p = torch.zeros(700, device=cuda, dtype=dtype, requires_grad=True)
    p.grad = torch.ones(700, device=cuda, dtype=dtype)
    p.grad[3] = value
    opt = optim.AdamW([p], state_bits=bits, weight_decay=0.0, max_grad_norm=1.0)
    opt.step()
    opt.step()
    q = torch.zeros(700, device=cuda, requires_grad=True)
    q.grad = p.grad.float()
    ref = torch.optim.AdamW([q], lr=1e-3, weight_decay=0.0)
    for _ in range(2):
        grad = q.grad.clone()
        torch.nn.utils.clip_grad_norm_([q], 1.0)
        ref.step()
        q.grad = grad
    assert torch.equal(p.isnan(), q.isnan())
    for name, tail in tails(opt, 700):
        assert bool((tail == 0).all()), name


@pytest.mark.parametrize("bits", [32, 8])
def test_loaded_state_has_zero_tails(cuda, bits):
    """Tails that something else filled are cleared by load_state_dict, the tensors' own values are the state's, and
    an optimiser takes its own state back as it is."""
    optim = pkg_module("optim")
    p = torch.randn(700, device=cuda).bfloat16().requires_grad_()
    p.grad = torch.randn(700, device=cuda).bfloat16()
    opt = optim.AdamW([p], state_bits=bits)
    opt.step()
    keep = {n: t.clone() for n, t in opt.state[p].items()}
    for name, flat in opt.state_buffers()[0].items():
        if name in ("exp_avg", "exp_avg_sq", "master"):
            flat[700:] = float("nan")
    opt.load_state_dict(opt.state_dict())
    for name, tail in tails(opt, 700):
        assert bool((tail == 0).all()), name
    for n, t in opt.state[p].items():
        assert torch.equal(t.float(), keep[n].float()), n
