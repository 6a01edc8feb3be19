"""layernorm.layer_norm of rows whose mean lies far above their spread, on a B200 against fp64.

Tolerances, in half steps H = 2^-24 of fp32.  The mean of a row is a sum with an error e; every centred value
d = x - mean - e has that error, and the mean of the d takes it out again.  What is left does not know the row's
mean any more, only D, the largest |x - mean| (e itself is far below D in these rows): d is off by 1 of D, the
mean of the d by its sum (at most 40 additions in a thread and 9 between threads) and its quotient (1), the
difference by 1: 52 of D.  The variance, a sum of 50 terms of two roundings, is off by 53 of itself, r by half of
that and the root's 4, at most 31; the products add 3: below 96 of D r |w| + |b|.  The backward pass repeats xh
from the stored mean, in two parts, and makes its sums the same way.
A constant row: e is a few units of the mean's last place, so d is a number of at most 6 bits, the same in every
column; the sum of up to 2^15 of them is exact, its quotient is d and the difference zero."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

H, K = 2.0 ** -24, 96
# a warp's lanes and less; a block a row in loads of 16 bytes, of two values, of one; rows read again
WIDTHS = [33, 184, 512, 1000, 1002, 4096, 8193, 9001, 12290, 20001]


def run(x, w, b, dy, eps=1e-5):
    ln = pkg_module("layernorm")
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = ln.layer_norm(*leaves, eps)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_constant_rows_give_the_bias(cuda, dim, dtype):
    g = torch.Generator(device=cuda).manual_seed(dim)
    rows = 200
    size = 10 ** (2 + 2.75 * torch.rand(rows, 1, device=cuda, generator=g))            # 1e2 to 5.6e4
    sign = torch.where(torch.rand(rows, 1, device=cuda, generator=g) < 0.5, -1.0, 1.0)
    x = (size * sign).to(dtype).expand(rows, dim).contiguous()
    w = torch.randn(dim, device=cuda, generator=g)
    b = torch.randn(dim, device=cuda, generator=g)
    y, dx, dw, db = run(x, w, b, torch.randn(rows, dim, device=cuda, generator=g).to(dtype))
    assert torch.equal(y, b.to(dtype).expand(rows, dim))
    assert bool((dw == 0).all())                                                        # xh is zero
    y = pkg_module("layernorm").layer_norm(x)
    assert bool((y == 0).all())


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("mean", [1e2, 1e4, -6e4])
def test_mean_far_above_the_spread(cuda, dim, mean):
    g = torch.Generator(device=cuda).manual_seed(dim)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g)
    rows = 50
    x, w, b, dy = rnd(rows, dim) + mean, 1 + 0.3 * rnd(dim), rnd(dim), rnd(rows, dim)
    y, dx, dw, db = run(x, w, b, dy)
    xd, wd, bd, dyd = (t.double() for t in (x, w, b, dy))
    c = xd - xd.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((c ** 2).mean(-1, keepdim=True) + 1e-5)
    xh, gr = c * r, dyd * wd
    m1, m2 = gr.mean(-1, keepdim=True), (gr * xh).mean(-1, keepdim=True)
    top = lambda t: t.abs().amax(-1, keepdim=True)
    off = K * H * top(c) * r
    want = {"y": xh * wd + bd, "dx": r * (gr - m1 - xh * m2), "dw": (dyd * xh).sum(0)}
    tol = {"y": off * wd.abs() + K * H * bd.abs(),
           "dx": r * (K * H * (top(gr) + top(xh) * top(gr * xh)) + off * (m2.abs() + top(xh) * top(gr))) + K * H * want["dx"].abs(),
           "dw": K * H * (dyd * xh).abs().sum(0) + (dyd.abs() * off).sum(0)}
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        worst = float(((got.double() - want[name]).abs() / tol[name]).max())
        assert worst <= 1, f"{name}: {worst:.3g} of the tolerance"


def test_small_spread_without_eps(cuda):
    """eps 0 and rows of two values one or two steps of the mean apart: half of the row each, so xh is -1 or 1. The
    centred values are numbers of 5 bits (the mean is off by 8 steps at most), their squares and the sums of 4,096 of
    them below 24 bits, the quotients exact: nothing is rounded before r.  y is off by
    the variance's 3 roundings, the root's 4 and the products' 3."""
    ln = pkg_module("layernorm")
    for dim in (64, 512, 4096):
        x = torch.full((40, dim), 1.0, device=cuda) * (1000.0 + torch.arange(40, device=cuda)[:, None])
        x[:, ::2] += 2.0 ** -13                        # the values' last place is 2^-14
        y = ln.layer_norm(x, eps=0.0)
        want = torch.ones_like(x)
        want[:, 1::2] = -1.0
        assert bool(((y - want).abs() <= 16 * H).all())
