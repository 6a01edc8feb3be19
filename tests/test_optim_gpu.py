"""optim.AdamW on a B200 against AdamW's formulas in fp64.

Tolerances: fp32 states are a fused product-sum each (under 4 half steps, 2^-24, of the terms' sizes, the
clip's scaling among them); a parameter's change is a quotient of those (under 32 half steps of
itself), and the subtraction rounds the parameter once (2 half steps with the decay's product).
16-bit parameters then are rounded: finfo(T).eps / 2.  8-bit moments are compared code by code with
a restatement of the stochastic rounding on uint64 in numpy, except where the number that decides lies
within 1e-4 of the border, which fp32 (off by 2^-20 of a code step, as values of 8 binades over
their block's scale) may see on the other side.
"""
import copy

import numpy as np
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

H = 2.0 ** -24
SHAPES = [(84, 512), (512,), (1,), (33, 7), (256,), (257,), (2048, 3), (5, 3, 11), (4100,)]


def make(cuda, dtype, seed=0, shapes=SHAPES, flat=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    params = []
    for i, s in enumerate(shapes):
        n = int(np.prod(s))
        if flat:                      # views at odd places: no alignment beyond the type's
            t = torch.zeros(n + 1 + i % 3, device=cuda, dtype=dtype)[1 + i % 3:].view(s)
            gr = torch.zeros(n + 1, device=cuda, dtype=dtype)[1:].view(s)
        else:
            t, gr = torch.zeros(s, device=cuda, dtype=dtype), torch.zeros(s, device=cuda, dtype=dtype)
        t.copy_(torch.randn(s, device=cuda, generator=g))
        gr.copy_(torch.randn(s, device=cuda, generator=g) * 10 ** (-3 + i % 4))
        t.requires_grad_()
        t.grad = gr
        params.append(t)
    return params


class Reference:
    """The formulas in fp64 on the values that the optimiser begins with."""

    def __init__(self, params, lr, betas, eps, wd, max_norm=None):
        self.p = [p.detach().double() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.t, self.args, self.max_norm = 0, (lr, betas, eps, wd), max_norm

    def step(self, grads):
        lr, (b1, b2), eps, wd = self.args
        self.t += 1
        norm = torch.sqrt(sum((g.double() ** 2).sum() for g in grads))
        c = 1.0 if self.max_norm is None else min(1.0, self.max_norm / (float(norm) + 1e-6))
        self.change = []
        for i, g in enumerate(grads):
            g = g.double() * c
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            ch = lr * self.m[i] / (1 - b1 ** self.t) / ((self.v[i] / (1 - b2 ** self.t)).sqrt() + eps)
            self.change.append(ch)
            self.p[i] = self.p[i] * (1 - lr * wd) - ch
        return norm


def close(got, want, tol, what):
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_against_fp64(cuda, dtype, flat, max_norm):
    """Five steps, new gradients each; 16-bit parameters through their masters."""
    opt_mod = pkg_module("optim")
    params = make(cuda, dtype, 1, flat=flat)
    args = (3e-3, (0.9, 0.999), 1e-6, 0.1)
    opt = opt_mod.AdamW(params, lr=args[0], betas=args[1], eps=args[2], weight_decay=args[3], max_grad_norm=max_norm)
    ref = Reference(params, *args, max_norm)
    g = torch.Generator(device=cuda).manual_seed(2)
    total = [torch.zeros_like(p) for p in ref.p]
    size_m, size_v = [torch.zeros_like(p) for p in ref.p], [torch.zeros_like(p) for p in ref.p]
    for k in range(5):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, device=cuda, generator=g) * 10.0 ** (k - 3))
        grads = [p.grad.clone() for p in params]
        norm = ref.step(grads)
        opt.step()
        c = 1.0 if max_norm is None else min(1.0, max_norm / (float(norm) + 1e-6))
        for i, p in enumerate(params):
            st = opt.state[p]
            gi = grads[i].double().abs() * c
            size_m[i] = 0.9 * size_m[i] + 0.1 * gi * 5
            size_v[i] = 0.999 * size_v[i] + 0.001 * gi ** 2 * 8
            close(st["exp_avg"], ref.m[i], 4 * H * size_m[i] + 1e-38, "exp_avg")
            close(st["exp_avg_sq"], ref.v[i], 4 * H * size_v[i] + 1e-38, "exp_avg_sq")
            # a moment near zero is off by its terms' roundings: its relative part enters the change
            lr, (b1, b2), eps, _ = args
            root = (ref.v[i] / (1 - b2 ** ref.t)).sqrt() + eps
            total[i] += lr * 4 * H * size_m[i] / (1 - b1 ** ref.t) / root + 32 * H * ref.change[i].abs() + 2 * H * ref.p[i].abs()
            fp32 = st["master"] if dtype != torch.float32 else p.detach()
            close(fp32, ref.p[i], total[i], "parameter")
            if dtype != torch.float32:
                assert torch.equal(p.detach(), fp32.to(dtype))
            assert int(st["step"]) == k + 1
            assert torch.equal(p.grad, grads[i])
        if max_norm is not None:
            assert abs(float(opt.grad_norm) - float(norm)) <= 64 * H * float(norm)


def test_equals_torch_adam_without_decay(cuda):
    """weight_decay 0 is torch.optim.Adam after clip_grad_norm_: within a few roundings over ten steps (each
    at most 64 half steps of a change of at most lr x 10)."""
    opt_mod = pkg_module("optim")
    a, b = make(cuda, torch.float32, 3), make(cuda, torch.float32, 3)
    mine = opt_mod.AdamW(a, lr=1e-3, eps=1e-5, weight_decay=0.0, max_grad_norm=0.5)
    ref = torch.optim.Adam(b, lr=1e-3, eps=1e-5)
    for _ in range(10):
        mine.step()
        torch.nn.utils.clip_grad_norm_([p for p in b], 0.5)
        ref.step()
        for p, q in zip(a, b):               # torch rescaled its gradients in place
            q.grad = p.grad.clone()
    for p, q in zip(a, b):
        assert bool(((p - q).abs() <= 10 * 64 * H * 1e-2 + 20 * H * q.abs()).all())


def test_without_masters(cuda):
    """16-bit parameters updated in fp32 and rounded: one step is the formula's, rounded to nearest."""
    opt_mod = pkg_module("optim")
    for dtype in (torch.bfloat16, torch.float16):
        params = make(cuda, dtype, 4)
        ref = Reference(params, 1e-2, (0.9, 0.99), 1e-6, 0.0)
        opt = opt_mod.AdamW(params, lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.0, master_weights=False)
        assert "master" not in opt.state[params[0]]
        grads = [p.grad.clone() for p in params]
        ref.step(grads)
        opt.step()
        half = torch.finfo(dtype).eps / 2
        for i, p in enumerate(params):
            close(p.detach(), ref.p[i], half * ref.p[i].abs() + 40 * H * (ref.change[i].abs() + ref.p[i].abs()) + 2.0 ** -25, "parameter")


def test_master_follows_a_parameter_set_from_outside(cuda):
    opt_mod = pkg_module("optim")
    p = torch.full((300,), 1.0, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    p.grad = torch.full_like(p, 1e-3)
    opt = opt_mod.AdamW([p], lr=1e-4, weight_decay=0.0)
    for _ in range(20):
        opt.step()
    # twenty changes of 1e-4 add up in the master (a bf16 step at 1.0 is 2^-8 below it)
    assert abs(float(opt.state[p]["master"][0]) - (1 - 20e-4)) < 1e-5
    with torch.no_grad():
        p[100:].fill_(3.0)
    opt.step()
    assert abs(float(opt.state[p]["master"][0]) - (1 - 21e-4)) < 1e-5
    assert abs(float(opt.state[p]["master"][200]) - (3 - 1e-4)) < 1e-5


# ---- 8-bit moments

def mix(z):
    with np.errstate(over="ignore"):
        z = z + np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return z ^ (z >> np.uint64(31))


def draws(seed, step, total):
    """16 random bits for each moment of each position."""
    key = mix(np.array([np.uint64(seed) ^ mix(np.array([step], dtype=np.uint64))[0]], dtype=np.uint64))
    pos = np.arange(total, dtype=np.uint64)
    with np.errstate(over="ignore"):
        word = mix(key + (pos >> np.uint64(1))) >> (np.uint64(32) * (pos & np.uint64(1)))
    return (word & np.uint64(0xFFFF)).astype(np.float64), ((word >> np.uint64(16)) & np.uint64(0xFFFF)).astype(np.float64)


def codes(values, bits, mant, low, most, floor):
    """(codes, scale, undecided) of fp64 values whose rounding `bits` (16 of them) decides."""
    v = values.reshape(-1, 256)
    scale = np.maximum(np.abs(v).max(1) / most, np.finfo(np.float32).tiny)
    a = np.minimum(np.abs(v) / scale[:, None], most).reshape(-1)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** low)))
    q = 2.0 ** (e - mant)
    x = a / q + bits / 65536
    c = np.floor(x) * q
    near = np.abs(x - np.round(x)) < 1e-4      # a power of two from either side as well: 16 - e + u or 8 + u of its steps
    if floor:
        c = np.where((a > 0) & (c == 0), 2.0 ** (low - mant), c)
    return np.copysign(c, values), scale, near


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("master", [False, True])
def test_eight_bit_codes(cuda, dtype, master):
    opt_mod = pkg_module("optim")
    seed, lr, b1, b2, eps = 77, 1e-3, 0.9, 0.999, 1e-6
    params = make(cuda, dtype, 5)
    opt = opt_mod.AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, state_bits=8, master_weights=master, seed=seed)
    buf = opt.state_buffers()[0]
    total = buf["exp_avg"].numel()
    assert buf["exp_avg"].dtype == torch.float8_e4m3fn and buf["exp_avg_sq"].dtype == torch.float8_e5m2
    g = torch.Generator(device=cuda).manual_seed(6)
    for t in range(1, 5):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, device=cuda, generator=g) * torch.exp(2 * torch.randn(p.shape, device=cuda, generator=g)) * 0.01)
        flat = lambda name: buf[name].double().cpu().numpy() * np.repeat(buf[name + "_scale"].double().cpu().numpy(), 256)
        grad, before = np.zeros(total), [p.detach().double() for p in params]
        if master and dtype != torch.float32:
            before = [opt.state[p]["master"].double().clone() if t > 1 else p.detach().double() for p in params]
        for p, at in zip(params, opt._buckets[0][0].firsts):
            grad[at:at + p.numel()] = p.grad.double().cpu().numpy().reshape(-1)
        m = b1 * flat("exp_avg") + (1 - b1) * grad
        v = b2 * flat("exp_avg_sq") + (1 - b2) * grad ** 2
        opt.step()
        um, uv = draws(seed, t, total)
        for name, val, u, mant, low, most, floor in (("exp_avg", m, um, 3, -6, 448.0, False), ("exp_avg_sq", v, uv, 2, -14, 57344.0, True)):
            want, scale, near = codes(val, u, mant, low, most, floor)
            got = buf[name].double().cpu().numpy()
            np.testing.assert_allclose(buf[name + "_scale"].double().cpu().numpy(), scale, rtol=8 * H)
            wrong = (got != want) & ~near
            assert not wrong.any(), f"{name}, step {t}: {wrong.sum()} codes differ, first at {np.nonzero(wrong)[0][0]}"
            assert near.mean() < 1e-2
        for i, (p, at) in enumerate(zip(params, opt._buckets[0][0].firsts)):
            cut = slice(at, at + p.numel())
            ch = lr * m[cut] / (1 - b1 ** t) / (np.sqrt(v[cut] / (1 - b2 ** t)) + eps)
            want = before[i] - torch.from_numpy(ch).to(cuda).view(p.shape)
            fp32 = opt.state[p]["master"] if master and dtype != torch.float32 else p.detach()
            half = torch.finfo(fp32.dtype).eps / 2
            # moments' terms of either sign: the change is off by 64 half steps of the largest one, lr x 10 x 4
            close(fp32, want, 64 * H * 40 * lr + (2 * H + half) * want.abs() + 2.0 ** -25, "parameter")


def test_eight_bit_rounding_is_unbiased(cuda):
    """The mean code of one gradient over many positions is the moment: 4096 blocks hold the same 256
    gradients; the mean over them of a code (a step at most apart, so a deviation of half a step at most)
    lies within 6 standard errors (6 x 0.5 / 64 of a step) of the value."""
    opt_mod = pkg_module("optim")
    base = torch.linspace(0.11, 0.9, 256, device=cuda)
    base[0] = 1.0                                                      # the scale
    p = torch.zeros(4096, 256, device=cuda, requires_grad=True)
    p.grad = base.expand(4096, 256).contiguous()
    opt = opt_mod.AdamW([p], state_bits=8, seed=9)
    opt.step()
    buf = opt.state_buffers()[0]
    for name, value, mant in (("exp_avg", 0.1 * base.double(), 3), ("exp_avg_sq", 1e-3 * base.double() ** 2, 2)):
        deq = buf[name].double().view(4096, 256) * buf[name + "_scale"].double()[:, None]
        scale = buf[name + "_scale"][0].double()
        step = 2.0 ** (torch.floor(torch.log2(value / scale)) - mant) * scale
        assert bool(((deq.mean(0) - value).abs() <= step * (6 * 0.5 / 64 + 1e-4)).all()), name


def test_eight_bit_special_values(cuda):
    """Zero gradients keep zero moments; a NaN or infinite gradient becomes a NaN of its own element and
    nothing else; tiny second moments stay above zero; tails past a tensor's end stay zero."""
    opt_mod = pkg_module("optim")
    p = torch.zeros(700, device=cuda, requires_grad=True)
    p.grad = torch.ones(700, device=cuda)
    p.grad[256:512] = 0.0
    p.grad[3], p.grad[4], p.grad[5] = float("nan"), float("inf"), 1e-12
    opt = opt_mod.AdamW([p], state_bits=8, weight_decay=0.0)
    opt.step()
    st, buf = opt.state[p], opt.state_buffers()[0]
    m, v = buf["exp_avg"].float(), buf["exp_avg_sq"].float()
    bad = torch.zeros(768, dtype=torch.bool, device=cuda)
    bad[3] = bad[4] = True
    assert torch.equal(m.isnan(), bad) and torch.equal(v.isnan(), bad)
    assert torch.equal(p.isnan(), bad[:700])
    assert float(v[5]) > 0 and bool((m[256:512] == 0).all()) and bool((p[256:512] == 0).all())
    assert bool((m[700:] == 0).all()) and bool((v[700:] == 0).all())
    assert st["exp_avg_scale"].shape == (3,) and bool(st["exp_avg_scale"].isfinite().all())


# ---- the optimiser around the step

@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_groups_and_counts(cuda, bits):
    """A tensor without a gradient keeps its value, state and count; groups have their own numbers; the
    clip is over all of them."""
    opt_mod = pkg_module("optim")
    a, b = make(cuda, torch.float32, 7), make(cuda, torch.bfloat16, 8)
    opt = opt_mod.AdamW([{"params": a, "lr": 1e-2}, {"params": b, "weight_decay": 0.5}], lr=1e-3, weight_decay=0.0,
                        state_bits=bits, max_grad_norm=1.0)
    keep = a[2].detach().clone()
    g2, a[2].grad = a[2].grad, None
    opt.step()
    norm = torch.sqrt(sum((p.grad.double() ** 2).sum() for p in a + b if p.grad is not None))
    assert abs(float(opt.grad_norm) - float(norm)) <= 64 * H * float(norm)
    assert torch.equal(a[2], keep) and int(opt.state[a[2]]["step"]) == 0 and int(opt.state[a[1]]["step"]) == 1
    a[2].grad = g2
    opt.step()
    assert int(opt.state[a[2]]["step"]) == 1 and int(opt.state[a[1]]["step"]) == 2
    for p in a + b:
        p.grad = None
    before = [p.detach().clone() for p in a + b]
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a + b, before)) and int(opt.state[a[1]]["step"]) == 2


def test_many_tensors(cuda):
    """More tensors than a launch's table holds (720), all but a few of one value: the same bits as the same
    tensors in two optimisers, and the norm over all of them."""
    opt_mod = pkg_module("optim")
    shapes = [(3,)] * 1500 + [(1000, 7)]
    a, b = make(cuda, torch.float32, 9, shapes), make(cuda, torch.float32, 9, shapes)
    one = opt_mod.AdamW(a, lr=1e-2)
    two = [opt_mod.AdamW(b[:700], lr=1e-2), opt_mod.AdamW(b[700:], lr=1e-2)]
    for _ in range(2):
        one.step()
        for o in two:
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert bool((one.state_buffers()[0]["step"] == 2).all())
    clipped = opt_mod.AdamW(a, lr=1e-2, max_grad_norm=0.1)
    clipped.step()
    norm = torch.sqrt(sum((p.grad.double() ** 2).sum() for p in a))
    assert abs(float(clipped.grad_norm) - float(norm)) <= 64 * H * float(norm)


def test_repeatable(cuda):
    opt_mod = pkg_module("optim")
    out = []
    for _ in range(2):
        params = make(cuda, torch.float32, 10, [(1000, 1000), (77,)])
        opt = opt_mod.AdamW(params, state_bits=8, max_grad_norm=0.3, seed=5)
        for _ in range(3):
            opt.step()
        out.append([*[p.detach() for p in params], *opt.state_buffers()[0].values(), opt.grad_norm])
    for x, y in zip(*out):
        assert torch.equal(x.view(torch.uint8) if x.dim() else x, y.view(torch.uint8) if y.dim() else y)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(cuda, bits):
    opt_mod = pkg_module("optim")
    a = make(cuda, torch.bfloat16, 11)
    opt = opt_mod.AdamW(a, lr=1e-2, state_bits=bits, seed=3)
    opt.step()
    b = [p.detach().clone().requires_grad_() for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    other = opt_mod.AdamW(b, lr=5.0, state_bits=bits, seed=3)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert other.param_groups[0]["lr"] == 1e-2
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for p, q in zip(a, b):
        assert int(other.state[q]["step"]) == 2
        for n in opt.state[p]:
            x, y = opt.state[p][n], other.state[q][n]
            assert torch.equal(x.float(), y.float())
    wrong = opt_mod.AdamW(b, state_bits=40 - bits)
    with pytest.raises(ValueError):
        wrong.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        opt_mod.AdamW(b[:2]).load_state_dict(opt.state_dict())
    with pytest.raises(TypeError):
        copy.deepcopy(opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts(cuda, bits):
    """Replays of a captured step equal as many eager steps, the clip and the step count among them; two graphs
    of two optimisers in turn do not disturb one another."""
    opt_mod = pkg_module("optim")
    sets = [make(cuda, torch.float32, s) for s in (12, 12, 13, 13)]
    opts = [opt_mod.AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=1.0) for ps in sets]
    for o in opts:
        o.step()
    graphs = []
    for o in (opts[0], opts[2]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o.step()
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        opts[1].step()
        opts[3].step()
    for a, b in ((0, 1), (2, 3)):
        assert all(torch.equal(p, q) for p, q in zip(sets[a], sets[b]))
        assert bool((opts[a].state_buffers()[0]["step"] == 4).all())
        assert torch.equal(opts[a].grad_norm, opts[b].grad_norm)


def test_two_optimisers_at_once(cuda):
    """Actor's and critic's steps on two streams: the bits of one after the other."""
    opt_mod = pkg_module("optim")
    sets = [make(cuda, torch.float32, s) for s in (14, 14, 15, 15)]
    opts = [opt_mod.AdamW(ps, lr=1e-2, state_bits=8, max_grad_norm=1.0) for ps in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, o in zip(streams, (opts[0], opts[2])):
            with torch.cuda.stream(st):
                o.step()
    torch.cuda.synchronize()
    for _ in range(5):
        opts[1].step()
        opts[3].step()
    for a, b in ((0, 1), (2, 3)):
        assert all(torch.equal(p, q) for p, q in zip(sets[a], sets[b]))


def test_writes_are_seen_by_autograd(cuda):
    """A step changes its parameters' versions, as torch's optimisers do: a backward pass over values saved
    before it refuses."""
    opt_mod = pkg_module("optim")
    p = torch.ones(8, device=cuda, requires_grad=True)
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt_mod.AdamW([p]).step()
    with pytest.raises(RuntimeError):
        y.backward()


def test_odd_gradients(cuda):
    """A gradient with strides of its own is taken as its values; an empty parameter is passed over."""
    opt_mod = pkg_module("optim")
    p, q = torch.ones(6, 4, device=cuda, requires_grad=True), torch.ones(6, 4, device=cuda, requires_grad=True)
    e = torch.zeros(0, 3, device=cuda, requires_grad=True)
    e.grad = torch.zeros(0, 3, device=cuda)
    g = torch.randn(4, 6, device=cuda)
    p.grad, q.grad = g.t(), g.t().contiguous()
    opt_mod.AdamW([p, e]).step()
    opt_mod.AdamW([q]).step()
    assert torch.equal(p, q)


def test_changed_parameters_are_refused(cuda):
    """Storage swapped for one of another size, type or layout is not written over; of the same form it is
    followed."""
    opt_mod = pkg_module("optim")
    for new in (torch.ones(9, 4, device=cuda), torch.ones(6, 4, device=cuda).half(), torch.ones(4, 6, device=cuda).t()):
        p = torch.ones(6, 4, device=cuda, requires_grad=True)
        p.grad = torch.ones_like(p)
        opt = opt_mod.AdamW([p])
        p.data = new
        with pytest.raises((RuntimeError, TypeError)):
            opt.step()
    p = torch.ones(6, 4, device=cuda, requires_grad=True)
    p.grad = torch.ones_like(p)
    opt = opt_mod.AdamW([p], lr=0.5, weight_decay=0.0)
    p.data = torch.full((6, 4), 3.0, device=cuda)
    opt.step()
    assert bool((p - 2.5).abs().max() < 1e-5)


def test_refusals(cuda):
    opt_mod = pkg_module("optim")
    p = torch.ones(4, 4, device=cuda, requires_grad=True)
    for kind, call in [
        (ValueError, lambda: opt_mod.AdamW([p], lr=-1.0)),
        (TypeError, lambda: opt_mod.AdamW([p], lr=torch.tensor(1.0))),
        (ValueError, lambda: opt_mod.AdamW([p], betas=(1.0, 0.9))),
        (ValueError, lambda: opt_mod.AdamW([p], eps=-1e-8)),
        (ValueError, lambda: opt_mod.AdamW([p], state_bits=16)),
        (ValueError, lambda: opt_mod.AdamW([p], max_grad_norm=0.0)),
        (ValueError, lambda: opt_mod.AdamW([torch.ones(3, requires_grad=True)])),
        (TypeError, lambda: opt_mod.AdamW([torch.ones(3, device=cuda, dtype=torch.float64, requires_grad=True)])),
        (ValueError, lambda: opt_mod.AdamW([torch.ones(3, 4, device=cuda).t().requires_grad_()])),
        (ValueError, lambda: opt_mod.AdamW([p, p])),
    ]:
        with pytest.raises(kind):
            call()


def test_update_of_the_trainer(cuda):
    """ppo_update with "adamw" (no decay) takes the steps that it takes with "adam": every parameter within
    Adam's own step of rounding (64 half steps of lr x 10 over 8 steps, plus what a different rounding of the
    parameters changes in the next gradients: 1e-5 of them as between split and plain products)."""
    tr = pkg_module("trainer")
    torch.manual_seed(0)
    base = tr.MLPActorCritic(hidden=(128, 128), activation="tanh").to(cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    T, n = 16, 64
    obs = torch.randn(T, n, 184, device=cuda, generator=g)
    act = torch.randint(0, 21, (T, n, 4), device=cuda, generator=g, dtype=torch.uint8)
    logp = torch.full((T, n), -12.0, device=cuda)
    val, adv, ret = (torch.randn(T, n, device=cuda, generator=g) for _ in range(3))
    out = {}
    for name in ("adam", "adamw"):
        model = copy.deepcopy(base)
        cfg = tr.PPOConfig(update_epochs=2, num_minibatches=4, target_kl=None, lr=1e-3, optimizer=name)
        opts = [tr.make_optimizer(ps, 1e-3, cfg) for ps in (model.actor_parameters(), model.critic_parameters())]
        assert isinstance(opts[0], pkg_module("optim").AdamW) == (name == "adamw")
        gen = torch.Generator(device=cuda).manual_seed(2)
        res = tr.ppo_update(model, *opts, cfg, obs, act, logp, val, adv, ret, generator=gen)
        out[name] = ([p.detach() for p in model.parameters()], res)
    for p, q in zip(*(out[k][0] for k in ("adam", "adamw"))):
        assert float((p - q).abs().max()) <= 2e-5
    for k in ("actor_grad_norm", "critic_grad_norm"):
        a, b = (float(out[n][1][k]) for n in ("adam", "adamw"))
        assert abs(a - b) <= 1e-4 * abs(a)
    with pytest.raises(ValueError):
        tr.make_optimizer(base.actor_parameters(), 1e-3, tr.PPOConfig(optimizer="sgd"))


def test_trainer_iteration(cuda):
    """PPOTrainer with 8-bit AdamW: rollout, update, the policy kernel's weights refreshed; finite throughout."""
    rl_env, tr, optim = pkg_module("rl_env"), pkg_module("trainer"), pkg_module("optim")
    env = rl_env.GpuDogfightVecEnv(256, substeps=6, seed=5)
    torch.manual_seed(5)
    cfg = tr.PPOConfig(rollout_steps=4, hidden=(128, 128), activation="tanh", update_epochs=2, num_minibatches=2,
                       target_kl=None, optimizer="adamw", weight_decay=1e-3, state_bits=8)
    t = tr.PPOTrainer(env, cfg, opponents=[tr.Opponent(tr.MLPActorCritic(hidden=(128, 128)).to(cuda))])
    assert isinstance(t.actor_opt, optim.AdamW) and isinstance(t.critic_opt, optim.AdamW)
    before = [p.detach().clone() for p in t.model.parameters()]
    res, _ = t.iteration()
    assert res["optimizer_steps"] == 4 and float(res["actor_grad_norm"]) > 0
    assert bool((t.actor_opt.state_buffers()[0]["step"] == 4).all())
    for p, q in zip(t.model.parameters(), before):
        assert bool(p.isfinite().all()) and not torch.equal(p, q)
