"""The gate's sigmoid in recurrence.gated_scan / gated_step on a B200, over all gates, against fp64.

Tolerances, in half steps H = 2^-24 of fp32: the exponential e (PTX: the hardware's 2^t is good to 2^-22, 4) with its
argument's remainder taken in by a fused product-sum (1) is off by 5; 1 / (1 + e) by e's 5, the sum's 1 and the
reciprocal's 2 (PTX: 2^-23): 8.  f is 1 - k where the gate is above zero, so k at most 1/2: 8 + 1; elsewhere it is
e k, with e at most 1: 5 + (5 / 2 + 1 + 2) + 1 = 11.5.  Both below 12 of themselves; what lies under 2^-126
may be zero."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

H = 2.0 ** -24
TINY = 2.0 ** -126


def gates(cuda, dtype):
    g = torch.Generator(device=cuda).manual_seed(1)
    return torch.cat([torch.linspace(-130, 130, 40001, device=cuda), torch.linspace(-20, 20, 20001, device=cuda),
                      4 * torch.randn(20000, device=cuda, generator=g)]).to(dtype)[None].contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_both_sides_to_their_own_last_places(cuda, dtype):
    """A state of 1 and x 0 leave f, a state of 0 and x 1 leave 1 - f; the state is fp32 whatever the inputs."""
    rec = pkg_module("recurrence")
    gate = gates(cuda, dtype)
    f, k = torch.ones(gate.shape, device=cuda), torch.zeros(gate.shape, device=cuda)
    rec.gated_step(gate, torch.zeros_like(gate), f)
    rec.gated_step(gate, torch.ones_like(gate), k)
    for got, want in ((f, torch.sigmoid(gate.double())), (k, torch.sigmoid(-gate.double()))):
        bad = (got.double() - want).abs() > 12 * H * want + TINY
        assert not bool(bad.any()), f"gates {gate[bad][:5].tolist()}"
    # the scan's pairs and single values: the same arithmetic
    for width in (gate.shape[1], gate.shape[1] - 1):
        g = gate[:, :width][None].contiguous()
        _, hn = rec.gated_scan(g, torch.zeros_like(g), torch.ones(1, width, device=cuda))
        assert torch.equal(hn, f[:, :width])


def test_gates_at_the_end_of_the_range(cuda):
    rec = pkg_module("recurrence")
    top = torch.finfo(torch.float32).max
    gate = torch.tensor([[float("inf"), top, 200.0, -200.0, -top, -float("inf"), float("nan")]], device=cuda)
    state = torch.full((1, 7), 3.0, device=cuda)
    h = rec.gated_step(gate, torch.full_like(gate, 5.0), state)
    assert torch.equal(h[:, :6], torch.tensor([[3.0, 3.0, 3.0, 5.0, 5.0, 5.0]], device=cuda)) and bool(h[:, 6:].isnan().all())
    low = torch.tensor([[torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max]], device=cuda, dtype=torch.bfloat16)
    state = torch.full((1, 2), 3.0, device=cuda)
    assert rec.gated_step(low, torch.full_like(low, 5.0), state).tolist() == [[5.0, 3.0]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("steps", [1, 3])
def test_gradients_on_both_sides(cuda, dtype, steps):
    """h0 1, x 0 and one gradient of 1 at the first step: dh0 is f, dx its 1 - f, dgate their product (a rounding of
    12 half steps each and two more), in the outputs' type; widths of pairs and of single values."""
    rec = pkg_module("recurrence")
    row = gates(cuda, dtype)
    for width in (row.shape[1], row.shape[1] - 1):
        gate = torch.zeros(steps, 1, width, device=cuda, dtype=dtype)
        gate[0] = row[:, :width]
        gate.requires_grad_()
        x = torch.zeros(steps, 1, width, device=cuda, dtype=dtype, requires_grad=True)
        h0 = torch.ones(1, width, device=cuda, requires_grad=True)
        h, _ = rec.gated_scan(gate, x, h0)
        dh = torch.zeros_like(h)
        dh[0] = 1
        dgate, dx, dh0 = torch.autograd.grad(h, (gate, x, h0), dh)
        f, k = torch.sigmoid(gate[0].detach().double()), torch.sigmoid(-gate[0].detach().double())
        half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        floor = TINY + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 0.0)
        for got, want, roundings, rounded in ((dh0, f, 12, 0.0), (dx[0], k, 12, half), (dgate[0], f * k, 26, half)):
            bound = (roundings * H * (1 + rounded) + rounded) * want + floor
            assert bool(((got.double() - want).abs() <= bound).all())
