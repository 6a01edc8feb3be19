"""Steady gates of recurrence.gated_scan on a B200 over long sequences, against fp64."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

H = 2.0 ** -24


# one sequence, whose time is cut into segments, and channels enough that it is not
@pytest.mark.parametrize("channels", [60, 74000])
def test_open_gates_keep_the_state(cuda, channels):
    """Gates of 18 to 40, the same at every step: 1 - f is at most 1.6e-8, below half a step under 1, so f rounds to 1
    and each step's error is 1 - f; products with 1 are exact. x is 0, so h_T = h_0 f^T and dh0 = dhn f^T: off by
    steps (1 - f) of themselves, and no more (the outputs' own rounding aside)."""
    rec = pkg_module("recurrence")
    steps = 16384 if channels < 1000 else 1500
    g = torch.linspace(18, 40, channels, device=cuda)
    k = torch.sigmoid(-g.double())
    gate = g.expand(steps, 1, channels)
    h0 = (1 + torch.rand(1, channels, device=cuda)).requires_grad_()
    x = torch.zeros(1, 1, 1, device=cuda).expand(steps, 1, channels)
    h, hn = rec.gated_scan(gate, x, h0)
    dhn = 1 + torch.rand(1, channels, device=cuda)
    dh0, = torch.autograd.grad(hn, h0, dhn)
    keep = torch.exp(steps * torch.log1p(-k))
    for got, first in ((hn.detach(), h0.detach()), (dh0, dhn)):
        want = first.double() * keep
        assert bool(((got.double() - want).abs() <= (steps * k * 1.01 + 2 * H) * first.double()).all())
