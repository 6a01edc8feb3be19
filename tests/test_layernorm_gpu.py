"""layernorm.layer_norm on a B200 against its formulas in fp64.

Tolerances: a value of type T is off by half a step, finfo(T).eps / 2 of itself, from its rounding; before
that everything is fp32.  The mean is a sum of D values made as at most 20 additions in a thread and
10 between threads: off by at most 30 half steps (2^-24) of the row's largest |x|.  The centred
value has that error and its own subtraction's, its square sum's relative error is twice as large
and halves again in the root; with the products that follow fewer than 64 half steps of
(max|x| r |w| + |b|).  The backward pass repeats xh (the same error) and two such means.  Column sums
add at most 64 terms in a chain (rows of a thread, warps of a block, partial sums of 32 threads).
"""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

H = 2.0 ** -24
K = 64


def reference(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    top = lambda t: t.abs().amax(-1, keepdim=True)
    off = K * H * top(x) * r                                    # of xh
    y = xh * w + b
    dx = r * (g - m1 - xh * m2)
    tol_y = off * w.abs() + K * H * b.abs()
    tol_dx = r * (K * H * (top(g) + top(xh) * top(g * xh)) + off * (m2.abs() + top(xh) * top(g))) + K * H * dx.abs()
    total = lambda t: t.reshape(-1, t.shape[-1]).sum(0)
    dw, db = total(dy * xh), total(dy)
    tol_dw = K * H * total((dy * xh).abs()) + total(dy.abs() * off)
    tol_db = K * H * total(dy.abs())
    return (y, dx, dw, db), (tol_y, tol_dx, tol_dw, tol_db)


def check(got, want, tol, name):
    half = torch.finfo(got.dtype).eps / 2
    # fp16 below its normal range steps by 2^-24
    bound = tol + half * want.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = (got.double() - want).abs() > bound
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() / bound.clamp_min(1e-300)).max()):.3g} of the tolerance"


def make(cuda, rows, dim, dtype, wdtype, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(rows, dim, device=cuda, generator=g) * (0.1 + 3 * torch.rand(rows, 1, device=cuda, generator=g))
    x = (x + 2 * torch.randn(rows, 1, device=cuda, generator=g)).to(dtype)
    w = b = None
    if wdtype is not None:
        w = (1 + 0.3 * torch.randn(dim, device=cuda, generator=g)).to(wdtype)
        b = torch.randn(dim, device=cuda, generator=g).to(wdtype)
    return x, w, b, torch.randn(rows, dim, device=cuda, generator=g).to(dtype)


def run(x, w, b, dy, eps=1e-5):
    ln = pkg_module("layernorm")
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    y = ln.layer_norm(next(it), *(next(it) if t is not None else None for t in (w, b)), eps)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    return (y.detach(), next(grads), *(next(grads) if t is not None else None for t in (w, b)))


# widths: one value; under a warp; odd; two to a load; vector tails; a block a row; the most that
# registers take and one above it; re-read rows
@pytest.mark.parametrize("dim", [1, 2, 3, 8, 17, 31, 33, 64, 184, 214, 215, 384, 512, 513, 1000, 1024, 2050, 4096, 4097,
                                 8192, 8193, 8200, 12288, 12289, 12290, 12296, 20001])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("rows", [1, 37])
def test_against_fp64(cuda, rows, dim, dtype, wdtype):
    x, w, b, dy = make(cuda, rows, dim, dtype, wdtype, 7 * rows + dim)
    want, tol = reference(x, w, b, dy, 1e-5)
    for got, v, t, name in zip(run(x, w, b, dy), want, tol, ("y", "dx", "dw", "db")):
        assert got.dtype == (wdtype if name in ("dw", "db") else dtype)
        check(got, v, t, name)


@pytest.mark.parametrize("rows,dim", [(4099, 184), (5000, 512), (4711, 7), (1500, 1536), (2000, 9000), (1700, 4097), (500, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(cuda, rows, dim, dtype):
    x, w, b, dy = make(cuda, rows, dim, dtype, torch.float32, rows)
    want, tol = reference(x, w, b, dy, 1e-5)
    first, second = run(x, w, b, dy), run(x, w, b, dy)
    for got, again, v, t, name in zip(first, second, want, tol, ("y", "dx", "dw", "db")):
        check(got, v, t, name)
        assert torch.equal(got, again), f"{name} differs between two runs"


def test_without_weight_or_bias(cuda):
    for use_w, use_b in ((False, False), (True, False), (False, True)):
        x, w, b, dy = make(cuda, 65, 200, torch.float32, torch.float32, 3)
        w, b = w if use_w else None, b if use_b else None
        want, tol = reference(x, w, b, dy, 1e-5)
        got = run(x, w, b, dy)
        for k, name in enumerate(("y", "dx", "dw", "db")):
            if got[k] is not None:
                check(got[k], want[k], tol[k], name)
        assert (got[2] is None) == (not use_w) and (got[3] is None) == (not use_b)


def test_layouts(cuda):
    """Leading axes, row strides (aligned and not), transposed and broadcast inputs and gradients."""
    ln = pkg_module("layernorm")
    g = torch.Generator(device=cuda).manual_seed(5)
    w = torch.randn(96, device=cuda, generator=g)
    big = torch.randn(40, 131, device=cuda, generator=g)
    cases = [torch.randn(3, 5, 7, 96, device=cuda, generator=g), big[:, 3:99], big[:, 4:100], big[::2, 1:97],
             torch.randn(96, 41, device=cuda, generator=g).t(), torch.randn(96, device=cuda, generator=g),
             torch.randn(1, 96, device=cuda, generator=g).expand(13, 96),
             torch.randn(6, 96, 5, device=cuda, generator=g).transpose(1, 2)]
    for x in cases:
        dy = torch.randn(x.shape, device=cuda, generator=g)
        want, tol = reference(x, w, None, dy, 1e-5)
        got = run(x, w, None, dy)
        for k, name in ((0, "y"), (1, "dx"), (2, "dw")):
            assert got[k].shape == want[k].shape
            check(got[k], want[k], tol[k], name)
    x = cases[0]
    leaf = x.detach().requires_grad_()
    one = torch.autograd.grad(ln.layer_norm(leaf, w).sum(), leaf)[0]        # dy broadcast with zero strides
    want, tol = reference(x, w, None, torch.ones_like(x), 1e-5)
    check(one, want[1], tol[1], "dx of a sum")


def test_rows_behind_the_last_are_left_alone(cuda):
    """The C entry writes rows x cols and nothing between or behind."""
    _lib = pkg_module("_lib")
    x = torch.randn(9, 100, device=cuda)
    y = torch.full((12, 104), 7.0, device=cuda)
    _lib.check(_lib.load().f16_layer_norm_fwd(_lib.ptr(x), 9, 100, 100, 2, None, None, 2, 1e-5, _lib.ptr(y), 104, None,
                                              None, _lib.stream_of(x)), "f16_layer_norm_fwd")
    assert bool((y[9:] == 7.0).all()) and bool((y[:, 100:] == 7.0).all())
    assert bool((y[:9, :100] != 7.0).all())


def test_special_values(cuda):
    """A constant row gives the bias (exactly: the centred values are zero), a NaN or infinite value
    makes its own row NaN and no other, eps is inside the root."""
    ln = pkg_module("layernorm")
    x = torch.randn(6, 130, device=cuda)
    x[1] = 3.25
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    b = torch.randn(130, device=cuda)
    y = ln.layer_norm(x, None, b)
    assert torch.equal(y[1], b)
    assert bool(y[2].isnan().all()) and bool(y[3].isnan().all())
    assert bool(y[[0, 1, 4, 5]].isfinite().all())
    far = torch.randn(4, 512, device=cuda) + 1e4                       # the mean far above the spread
    want, tol = reference(far, None, None, torch.ones_like(far), 1e-5)
    check(ln.layer_norm(far), want[0], tol[0], "y")
    want, tol = reference(far, None, None, torch.ones_like(far), 100.0)
    check(ln.layer_norm(far, eps=100.0), want[0], tol[0], "y")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_cancels(cuda, dtype):
    """A row of one value has no gradient, exactly; of rows of two (xh = +-1 but for eps) the gradient is what
    remains of much larger terms. In half steps H of fp32, with d = x - mu and q = |mu| / |d|: mu is rounded
    once, d is off by q + 1 of itself; in the variance the mean's part cancels to second order, which leaves
    2 + 1 + 1 and 1 for eps, so r is off by 2.5 and its own 4, at most 7, and xh by q + 9. g is off by 1, m1 by
    2, m2 by q + 12, xh m2 by 2 q + 22, the two sums add 2 of at most 2 terms' size each, and r with its product
    8 more: below 2 q + 40 of r max|g|, and twice the q for its second order."""
    x, w, b, dy = make(cuda, 300, 1, dtype, torch.float32, 1)
    y, dx, dw, db = run(x, w, b, dy)
    assert bool((dx == 0).all()) and bool((dw == 0).all()) and torch.equal(y, b.to(dtype).expand(300, 1))
    x, w, b, dy = make(cuda, 300, 2, dtype, torch.float32, 2)
    want, _ = reference(x, w, b, dy, 1e-5)
    got = run(x, w, b, dy)[1]
    r = 1 / torch.sqrt(x.double().var(-1, unbiased=False, keepdim=True) + 1e-5)
    mu = x.double().mean(-1, keepdim=True)
    q = mu.abs() / (x.double() - mu).abs().amax(-1, keepdim=True).clamp_min(1e-300)
    size = r * (dy.double() * w.double()).abs().amax(-1, keepdim=True)
    half = torch.finfo(dtype).eps / 2
    assert bool(((got.double() - want[1]).abs() <= (4 * q + 40) * H * size + half * want[1].abs()).all())


def test_empty(cuda):
    ln = pkg_module("layernorm")
    x = torch.zeros(0, 5, device=cuda, requires_grad=True)
    w, b = torch.ones(5, device=cuda, requires_grad=True), torch.ones(5, device=cuda, requires_grad=True)
    y = ln.layer_norm(x, w, b)
    y.sum().backward()
    assert y.shape == (0, 5) and x.grad.shape == (0, 5)
    assert torch.equal(w.grad, torch.zeros(5, device=cuda)) and torch.equal(b.grad, w.grad)


def test_gradient_against_differences(cuda):
    """Central differences of a fp32 loss: step 2^-6 on values of size 1, so the difference quotient's
    rounding (a sum of 51 terms of size 1: 51 x 2^-24 / 2^-5) and the cubic term (2^-12 of third
    derivatives of a few units) both stay under 1e-3 of the gradients' largest."""
    ln = pkg_module("layernorm")
    g = torch.Generator(device=cuda).manual_seed(11)
    x = torch.randn(3, 17, device=cuda, generator=g, requires_grad=True)
    w = (1 + 0.1 * torch.randn(17, device=cuda, generator=g)).requires_grad_()
    c = torch.randn(3, 17, device=cuda, generator=g)
    loss = lambda x, w: float((ln.layer_norm(x, w).double() * c).sum())
    gx, gw = torch.autograd.grad((ln.layer_norm(x, w) * c).sum(), (x, w))
    h = 2.0 ** -6
    with torch.no_grad():
        for t, grad in ((x, gx), (w, gw)):
            flat = t.view(-1)
            for i in range(0, flat.numel(), 5):
                old = float(flat[i])
                flat[i] = old + h
                up = loss(x, w)
                flat[i] = old - h
                down = loss(x, w)
                flat[i] = old
                assert abs((up - down) / (2 * h) - float(grad.view(-1)[i])) <= 1e-3 * float(grad.abs().max()) + 4e-3


def test_streams_and_graph(cuda):
    """On a side stream, and forward and backward captured into a graph and replayed on new data."""
    ln = pkg_module("layernorm")
    x = torch.randn(70, 300, device=cuda)
    w = torch.randn(300, device=cuda)
    want = ln.layer_norm(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ln.layer_norm(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs, ws, dy = x.clone().requires_grad_(), w.clone().requires_grad_(), torch.randn_like(x)

    def both():
        y = ln.layer_norm(xs, ws)
        return (y, *torch.autograd.grad(y, (xs, ws), dy))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [t.detach() for t in both()]
    with torch.no_grad():
        xs.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, both()):
        assert torch.equal(a, b.detach())


def test_module_and_tower(cuda):
    """LayerNorm is torch's module with the same parameters, and run_tower keeps the Linear before it on
    the split path: the tower against fp64 at the split path's own tolerance (1e-5)."""
    ln, sm = pkg_module("layernorm"), pkg_module("splitmm")
    torch.manual_seed(2)
    net = torch.nn.Sequential(torch.nn.Linear(184, 256), ln.LayerNorm(256), torch.nn.Tanh(), torch.nn.Linear(256, 84)).to(cuda)
    ref = torch.nn.Sequential(torch.nn.Linear(184, 256), torch.nn.LayerNorm(256), torch.nn.Tanh(),
                              torch.nn.Linear(256, 84)).double().to(cuda)
    ref.load_state_dict({k: v.double() for k, v in net.state_dict().items()})
    x, dy = torch.randn(3000, 184, device=cuda), torch.randn(3000, 84, device=cuda)
    y = sm.run_tower(net, x)
    names = {n.name() for n in _nodes(y.grad_fn)}
    assert any("SplitBlock" in n for n in names) and any("_LayerNorm" in n for n in names)
    y.backward(dy)
    z = ref(x.double())
    z.backward(dy.double())
    rel = lambda a, b: float((a.double() - b).abs().max() / b.abs().max())
    assert rel(y.detach(), z.detach()) <= 1e-5
    for p, q in zip(net.parameters(), ref.parameters()):
        assert rel(p.grad, q.grad) <= 1e-5


def _nodes(fn, seen=None):
    seen = set() if seen is None else seen
    if fn is not None and fn not in seen:
        seen.add(fn)
        for f, _ in fn.next_functions:
            _nodes(f, seen)
    return seen


def test_refusals(cuda):
    ln = pkg_module("layernorm")
    x = torch.randn(4, 8, device=cuda)
    with pytest.raises(TypeError):
        ln.layer_norm(x.double())
    with pytest.raises(TypeError):
        ln.layer_norm(x, torch.ones(8, device=cuda, dtype=torch.float16))
    with pytest.raises(TypeError):
        ln.layer_norm(x.half(), torch.ones(8, device=cuda), torch.ones(8, device=cuda, dtype=torch.float16))
    with pytest.raises(ValueError):
        ln.layer_norm(x, torch.ones(7, device=cuda))
    with pytest.raises(ValueError):
        ln.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError):
        ln.layer_norm(x[0, 0])
    with pytest.raises(ValueError):
        ln.layer_norm(x[:, :0])
    with pytest.raises(ValueError):
        ln.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        ln.LayerNorm(8).to(cuda)(x[:, :4])
