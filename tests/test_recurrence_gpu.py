"""recurrence.gated_scan / linear_scan / *_step on a B200 against the recurrence in fp64, step by step.

Tolerances: the fp32 recurrence makes at each step an error of at most C half steps (2^-24) of
|a_t h_{t-1}| + |b_t|, and multiplies the error before it by |a_t|; `errors` runs that bound beside the fp64
states.  C counts the roundings of a step: a product, an addition, and the coefficients, of which
the gate's exponential is the largest (its argument's rounding: 2 + 1.2 |gate| units, i.e. under 26
half steps for |gate| <= 8, and twice more in f and 1 - f).  Joining chunks multiplies the steps'
coefficients first, which rounds once more per step.  C = 96 covers all of it.  The gradient's
recurrence is bounded the same way, with the states' bound on top; the product that makes dgate
adds 8 C.  A value of type T then is off by its rounding, finfo(T).eps / 2 of itself.
"""
import ctypes

import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu

H, C = 2.0 ** -24, 96


def make(cuda, steps, batch, dim, dtype, gated, seed, resets=False, padded=False, initial=True, batch_first=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    shape = (batch, steps, dim) if batch_first else (steps, batch, dim)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g)
    gate = (rnd(*shape) + 2).clamp(-8, 8)
    if not gated:
        gate = torch.sigmoid(gate) * torch.where(torch.rand(*shape, device=cuda, generator=g) < 0.2, -1.0, 1.0)
    tr = lambda t: t.to(dtype).transpose(0, 1) if batch_first else t.to(dtype)
    d = dict(gate=tr(gate), x=tr(rnd(*shape)), h0=rnd(batch, dim) if initial else None,
             reset=torch.rand(steps, batch, device=cuda, generator=g) < 0.1 if resets else None, lengths=None)
    if padded:
        d["lengths"] = torch.randint(0, steps + 1, (batch,), device=cuda, generator=g)
        d["lengths"][0] = 0
        d["lengths"][-1] = steps
    return d, tr(rnd(*shape)), rnd(batch, dim)


def reference(d, gated, dh, dhn):
    """(values, bounds) of h, hn, dgate, dx, dh0 in fp64."""
    gate, x = d["gate"].double(), d["x"].double()
    steps, batch, dim = x.shape
    f = torch.sigmoid(gate) if gated else gate
    k = torch.sigmoid(-gate) if gated else torch.ones_like(gate)
    h = torch.zeros(batch, dim, dtype=torch.float64, device=x.device) if d["h0"] is None else d["h0"].double()
    dh, dhn = dh.double(), dhn.double()
    cut = torch.zeros(steps, batch, 1, dtype=torch.bool, device=x.device) if d["reset"] is None else d["reset"].bool().unsqueeze(2)
    live = torch.ones_like(cut)
    if d["lengths"] is not None:
        live = (torch.arange(steps, device=x.device)[:, None] < d["lengths"][None]).unsqueeze(2)
    e = torch.zeros_like(h)
    hs, es, before, ebefore = [], [], [], []
    zero = torch.zeros_like(h)
    for t in range(steps):
        hp, ep = torch.where(cut[t], zero, h), torch.where(cut[t], zero, e)
        b = torch.where(live[t], k[t] * x[t], zero)
        new = f[t] * hp + b
        enew = f[t].abs() * ep + C * H * ((f[t] * hp).abs() + b.abs())
        before.append(hp); ebefore.append(ep)
        h, e = torch.where(live[t], new, h), torch.where(live[t], enew, e)
        hs.append(torch.where(live[t], h, zero)); es.append(e)
    out = {"h": torch.stack(hs), "hn": h}
    tol = {"h": torch.stack(es), "hn": e}
    G, E = dhn, torch.zeros_like(h)
    dg, dx, tg, tx = [], [], [], []
    for t in reversed(range(steps)):
        Gt = torch.where(live[t], dh[t] + G, G)
        Et = E + C * H * torch.where(live[t], dh[t].abs() + G.abs(), zero)
        back = f[t] * k[t] if gated else torch.ones_like(f[t])
        diff = before[t] - x[t] if gated else before[t]
        size = before[t].abs() + x[t].abs() if gated else before[t].abs()
        dg.append(torch.where(live[t], Gt * diff * back, zero))
        tg.append(back * (Et * diff.abs() + Gt.abs() * ebefore[t] + 8 * C * H * Gt.abs() * size))
        dx.append(torch.where(live[t], Gt * k[t], zero))
        tx.append(k[t] * (Et + C * H * Gt.abs()))
        nextG = torch.where(cut[t], zero, f[t] * Gt)
        nextE = torch.where(cut[t], zero, f[t].abs() * Et + C * H * (f[t] * Gt).abs())
        G, E = torch.where(live[t], nextG, Gt), torch.where(live[t], nextE, E)
    for name, v, w in (("dgate", dg, tg), ("dx", dx, tx)):
        out[name], tol[name] = torch.stack(v[::-1]), torch.stack(w[::-1])
    out["dh0"], tol["dh0"] = G, E
    return out, tol


def run(d, gated, dh, dhn):
    rec = pkg_module("recurrence")
    leaves = {n: d[n].detach().requires_grad_() for n in ("gate", "x", "h0") if d[n] is not None}
    h, hn = (rec.gated_scan if gated else rec.linear_scan)(leaves["gate"], leaves["x"], leaves.get("h0"),
                                                           reset=d["reset"], lengths=d["lengths"])
    grads = torch.autograd.grad((h, hn), list(leaves.values()), (dh, dhn))
    return {"h": h.detach(), "hn": hn.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def check(got, want, tol, names=None):
    for name in names or got:
        a, w = got[name].double(), want[name]
        half = torch.finfo(got[name].dtype).eps / 2
        bound = tol[name] * (1 + half) + half * w.abs() + (2.0 ** -25 if got[name].dtype == torch.float16 else 1e-37)
        bad = (a - w).abs() > bound
        assert a.shape == w.shape and bool(a.isfinite().all())
        assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(((a - w).abs() / bound).max()):.3g} of the tolerance"


# one step; below, at and above a chunk of 16; several chunks; warps of a block; blocks of a cluster; more
# than one tile of a cluster (2,048 steps)
@pytest.mark.parametrize("steps", [1, 2, 15, 16, 17, 40, 256, 300, 2100, 4500])
@pytest.mark.parametrize("batch,dim", [(1, 1), (2, 66), (3, 185)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gated", [True, False])
def test_against_fp64(cuda, steps, batch, dim, dtype, gated):
    every = steps in (17, 300, 2100)
    d, dh, dhn = make(cuda, steps, batch, dim, dtype, gated, steps + dim, resets=every, padded=every and batch > 1,
                      initial=steps != 16, batch_first=steps in (40, 300))
    got = run(d, gated, dh, dhn)
    want, tol = reference(d, gated, dh, dhn)
    check(got, want, tol)


@pytest.mark.parametrize("batch,dim", [(1024, 96), (1500, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [True, False])
def test_many_channels(cuda, batch, dim, dtype, gated):
    d, dh, dhn = make(cuda, 50, batch, dim, dtype, gated, dim, resets=True, padded=True)
    got, again = run(d, gated, dh, dhn), run(d, gated, dh, dhn)
    want, tol = reference(d, gated, dh, dhn)
    check(got, want, tol)
    for n in got:
        assert torch.equal(got[n], again[n])


@pytest.mark.parametrize("steps,batch,dim", [(100, 4, 64), (30, 3000, 64)])
def test_reset_types_and_strides(cuda, steps, batch, dim):
    """bool, uint8 and fp32 flags give the same bits, as do strides along time and batch; an input off the
    alignment of pairs takes other kernels (and cuts time elsewhere), within the tolerance."""
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, steps, batch, dim, torch.bfloat16, True, 5, resets=True)
    want = run(d, True, dh, dhn)
    for kind in (torch.uint8, torch.float32):
        got = run({**d, "reset": d["reset"].to(kind)}, True, dh, dhn)
        assert all(torch.equal(got[n], want[n]) for n in want)
    flipped = d["reset"].t().contiguous().t()
    wide = torch.zeros(steps, batch, dim + 3, device=cuda, dtype=torch.bfloat16)
    odd = wide[:, :, 1:dim + 1]                              # off every alignment
    odd.copy_(d["x"])
    two = torch.zeros(2 * steps, batch, dim, device=cuda, dtype=torch.bfloat16)
    two[::2] = d["gate"]
    dhs = dh.transpose(0, 1).contiguous().transpose(0, 1)
    got = run({**d, "reset": flipped, "gate": two[::2]}, True, dhs, dhn)
    assert all(torch.equal(got[n], want[n]) for n in want)
    ref, tol = reference(d, True, dh, dhn)
    check(run({**d, "x": odd}, True, dh, dhn), ref, tol)
    h, _ = rec.gated_scan(d["gate"].transpose(0, 1).contiguous().transpose(0, 1),
                          d["x"].transpose(0, 1).contiguous().transpose(0, 1), d["h0"], reset=d["reset"])
    assert torch.equal(h, want["h"]) and h.stride(0) < h.stride(1)      # batch-first in, batch-first out


@pytest.mark.parametrize("steps,batch,dim", [(700, 2, 32), (40, 2500, 64)])
@pytest.mark.parametrize("gated", [True, False])
def test_what_is_masked_does_not_leak(cuda, steps, batch, dim, gated):
    """NaN and infinities behind a sequence's length, and a state made infinite or NaN before a reset,
    leave the rest as it is: the run with them equals the run without, where they do not belong."""
    d, dh, dhn = make(cuda, steps, batch, dim, torch.float32, gated, 9)
    cut = steps // 2
    d["reset"] = torch.zeros(steps, batch, device=cuda, dtype=torch.bool)
    d["reset"][cut] = True
    d["lengths"] = torch.full((batch,), steps - 7, device=cuda)
    want = run(d, gated, dh, dhn)
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min):
        for name in ("x", "gate"):
            e = {**d, name: d[name].clone()}
            e[name][steps - 7:] = value
            dirty = dh.clone()
            dirty[steps - 7:] = value
            got = run(e, gated, dirty, dhn)
            assert all(torch.equal(got[n], want[n]) for n in want)
        bad = {**d, "x": d["x"].clone()}
        bad["x"][3] = value
        got = run(bad, gated, dh, dhn)
        assert torch.equal(got["h"][cut:], want["h"][cut:]) and torch.equal(got["hn"], want["hn"])
        assert torch.equal(got["dgate"][cut:], want["dgate"][cut:])
        assert torch.equal(got["dx"], want["dx"])                      # does not depend on x
    assert bool((want["h"][steps - 7:] == 0).all()) and bool((want["dx"][steps - 7:] == 0).all())


def test_empty_sequences_and_clamped_lengths(cuda):
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, 20, 3, 8, torch.float32, True, 1)
    d["lengths"] = torch.tensor([0, -5, 99], device=cuda)
    got = run(d, True, dh, dhn)
    want, tol = reference({**d, "lengths": torch.tensor([0, 0, 20], device=cuda)}, True, dh, dhn)
    check(got, want, tol)
    assert torch.equal(got["hn"][:2], d["h0"][:2]) and torch.equal(got["dh0"][:2], dhn[:2])
    for shape in ((0, 3, 8), (5, 0, 8), (5, 3, 0)):
        z = torch.zeros(shape, device=cuda, requires_grad=True)
        h0 = torch.ones(shape[1:], device=cuda, requires_grad=True)
        h, hn = rec.gated_scan(z, z, h0)
        assert h.shape == shape and torch.equal(hn, h0)
        (h.sum() + 2 * hn.sum()).backward()
        assert torch.equal(h0.grad, torch.full(shape[1:], 2.0, device=cuda))


def test_partial_gradients(cuda):
    """Only some inputs require a gradient, only one output is used, inputs are broadcast."""
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, 70, 4, 12, torch.float32, True, 2)
    zero_h, zero_n = torch.zeros_like(dh), torch.zeros_like(dhn)
    x = d["x"].detach().requires_grad_()
    h, hn = rec.gated_scan(d["gate"], x, d["h0"])
    want, tol = reference(d, True, dh, zero_n)
    check({"dx": torch.autograd.grad(h, x, dh)[0]}, want, tol)
    h, hn = rec.gated_scan(d["gate"], x, d["h0"])
    want, tol = reference(d, True, zero_h, dhn)
    check({"dx": torch.autograd.grad(hn, x, dhn)[0]}, want, tol)
    row = torch.randn(12, device=cuda, requires_grad=True)               # one gate for all steps and sequences
    h, hn = rec.gated_scan(row.expand(70, 4, 12), d["x"], d["h0"])
    got = torch.autograd.grad(h, row, dh)[0]
    e = {**d, "gate": row.detach().expand(70, 4, 12)}
    want, tol = reference(e, True, dh, zero_n)
    total = want["dgate"].sum((0, 1))
    assert bool(((got.double() - total).abs() <= tol["dgate"].sum((0, 1)) + 280 * H * want["dgate"].abs().sum((0, 1))).all())


# several sequences to a warp, with widths that fit 16-byte copies (8, 16, 24), that do not (5, 14), and more
# sequences than a ballot has halves for (1, 2)
@pytest.mark.parametrize("batch,dim", [(75, 1), (70, 2), (40, 5), (33, 8), (21, 14), (70, 16), (9, 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [True, False])
def test_sequences_that_share_a_warp(cuda, batch, dim, dtype, gated):
    for steps, batch_first in ((50, False), (333, True)):
        d, dh, dhn = make(cuda, steps, batch, dim, dtype, gated, dim, resets=True, padded=True, batch_first=batch_first)
        want, tol = reference(d, gated, dh, dhn)
        check(run(d, gated, dh, dhn), want, tol)


def call(entry, d, gated, scratch, **buffers):
    """A C entry on time-major fp32 tensors, with the scratch given (None: time is not cut)."""
    _lib = pkg_module("_lib")
    rec = pkg_module("recurrence")
    b = {**dict.fromkeys(("h", "hn", "saved", "dh", "dhn", "dgate", "dx", "dh0")), **buffers}
    a = rec._args(d["gate"], d["x"], d["h0"], d["reset"], d["lengths"], int(gated), b["h"], b["hn"], b["saved"],
                  (scratch, 0 if scratch is None else scratch.numel()), b["dh"], b["dhn"], b["dgate"], b["dx"], b["dh0"])
    _lib.check(getattr(_lib.load(), entry)(ctypes.byref(a), _lib.stream_of(d["x"])), entry)


@pytest.mark.parametrize("steps,batch,dim", [(5000, 3, 7), (600_000, 1, 1)])
def test_cut_and_uncut_time(cuda, steps, batch, dim):
    """With scratch time is cut into segments (600,000 steps: more than the 1,024 whose states are joined at a
    time), without it is not: both are within the bound of the recurrence, so within twice the bound of each
    other.  The bound of |a| <= 0.9: errors of C half steps a step add up to at most C H (|a h| + |x|) / 0.1."""
    _lib = pkg_module("_lib")
    g = torch.Generator(device=cuda).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g)
    d = dict(gate=rnd(steps, batch, dim).clamp(-0.9, 0.9), x=rnd(steps, batch, dim), h0=rnd(batch, dim),
             reset=torch.rand(steps, batch, device=cuda, generator=g) < 0.01, lengths=None)
    dh, dhn = rnd(steps, batch, dim), rnd(batch, dim)
    n = _lib.load().f16_scan_scratch_floats(steps, batch, dim)
    assert n > 0
    out = []
    for scratch in (None, torch.empty(n, device=cuda), torch.empty(n - 1, device=cuda)):
        saved = torch.empty(_lib.load().f16_scan_saved_floats(steps, batch, dim), device=cuda)
        o = dict(h=torch.empty_like(d["x"]), hn=torch.empty(batch, dim, device=cuda))
        call("f16_scan_fwd", d, False, scratch, saved=saved, **o)
        q = dict(dgate=torch.empty_like(dh), dx=torch.empty_like(dh), dh0=torch.empty(batch, dim, device=cuda))
        call("f16_scan_bwd", d, False, scratch, saved=saved, dh=dh, dhn=dhn, **q)
        out.append({**o, **q})
    top = {"h": 1.0, "hn": 1.0, "dx": 1.0, "dh0": 1.0, "dgate": float(out[0]["h"].abs().max())}
    for name, v in out[0].items():
        bound = 4 * C * H * 10 * (float(v.abs().max()) + top[name] * float(d["x"].abs().max()))
        assert float((v - out[1][name]).abs().max()) <= bound, name
        assert torch.equal(v, out[2][name])                # too little scratch: as without


def test_two_scans_at_once(cuda):
    """On two streams, each with scratch of its own: the bits of one after the other."""
    cases = [make(cuda, 3000, 2, 40, torch.bfloat16, True, s, resets=True) for s in (1, 2)]
    want = [run(d, True, dh, dhn) for d, dh, dhn in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, (d, dh, dhn) in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(run(d, True, dh, dhn))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[n], b[n]) for n in b)


def test_no_gradient_saves_no_states(cuda):
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, 33, 5, 20, torch.bfloat16, True, 4)
    with torch.no_grad():
        h, hn = rec.gated_scan(d["gate"], d["x"], d["h0"])
    full = run(d, True, dh, dhn)
    assert torch.equal(h, full["h"]) and torch.equal(hn, full["hn"])


def test_gradient_against_differences(cuda):
    """Central differences in every input of a short scan: steps of 2^-7, under 2^-14 of third derivatives
    and 2^-24 x 60 terms / 2^-6 of rounding: 2e-3."""
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, 6, 1, 5, torch.float32, True, 8)
    d["reset"] = torch.zeros(6, 1, device=cuda, dtype=torch.bool)
    d["reset"][3] = True
    got = run(d, True, dh, dhn)

    def loss():
        h, hn = rec.gated_scan(d["gate"], d["x"], d["h0"], reset=d["reset"])
        return float((h.double() * dh).sum() + (hn.double() * dhn).sum())

    e = 2.0 ** -7
    for name in ("gate", "x", "h0"):
        flat, grad = d[name].view(-1), got["d" + name].view(-1)
        for i in range(flat.numel()):
            old = float(flat[i])
            flat[i] = old + e
            up = loss()
            flat[i] = old - e
            down = loss()
            flat[i] = old
            assert abs((up - down) / (2 * e) - float(grad[i])) <= 2e-3


@pytest.mark.parametrize("batch,dim", [(1, 1), (7, 185), (256, 512), (33, 12)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gated", [True, False])
def test_steps_equal_the_scan(cuda, batch, dim, dtype, gated):
    """A decision at a time gives the sequence's states: the step's arithmetic is the walking scan's, so
    within the scan's tolerance of fp64."""
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, 9, batch, dim, dtype, gated, 3, resets=True)
    want, tol = reference(d, gated, dh, dhn)
    state = d["h0"].clone()
    version = state._version
    hs = [(rec.gated_step if gated else rec.linear_step)(d["gate"][t], d["x"][t], state, reset=d["reset"][t])
          for t in range(9)]
    check({"h": torch.stack(hs), "hn": state}, want, tol)
    assert state._version > version


def test_step_layouts(cuda):
    rec = pkg_module("recurrence")
    for dtype in (torch.float32, torch.bfloat16):
        g, x = torch.randn(6, 40, device=cuda).to(dtype), torch.randn(6, 40, device=cuda).to(dtype)
        h = torch.randn(6, 40, device=cuda)
        state = h.clone()
        want = rec.gated_step(g, x, state)
        pool = torch.full((8, 44), 5.0, device=cuda)
        pool[1:7, :40] = h
        out = torch.full((6, 48), 5.0, device=cuda, dtype=dtype)
        flags = torch.zeros(6, 2, device=cuda)[:, 0]
        got = rec.gated_step(g.t().contiguous().t(), x, pool[1:7, :40], reset=flags, out=out[:, :40])
        assert torch.equal(got, want) and torch.equal(pool[1:7, :40], state)
        assert bool((pool[0] == 5).all()) and bool((pool[:, 40:] == 5).all()) and bool((out[:, 40:] == 5).all())
        state = torch.full((6, 40), float("nan"), device=cuda)
        fresh = rec.gated_step(g, x, state, reset=torch.ones(6, device=cuda, dtype=torch.bool))
        assert bool(fresh.isfinite().all())
        assert rec.gated_step(g[:0], x[:0], h[:0]).shape == (0, 40)


def test_streams_and_graph(cuda):
    """Both forms on a side stream, and captured: forward and backward of a split scan, and a decision whose
    state advances with every replay."""
    rec = pkg_module("recurrence")
    d, dh, dhn = make(cuda, 600, 2, 64, torch.bfloat16, True, 6, resets=True)
    want = run(d, True, dh, dhn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(d, True, dh, dhn)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(d, True, dh, dhn)
    d["x"].copy_(torch.randn(d["x"].shape, device=cuda))
    graph.replay()
    fresh = run(d, True, dh, dhn)
    assert all(torch.equal(held[n], fresh[n]) for n in fresh)
    state, ref = torch.zeros(2, 64, device=cuda), torch.zeros(2, 64, device=cuda)
    step = torch.cuda.CUDAGraph()
    with torch.cuda.graph(step):
        out = rec.gated_step(d["gate"][0], d["x"][0], state)
    state.zero_()
    for _ in range(3):
        step.replay()
        want_out = rec.gated_step(d["gate"][0], d["x"][0], ref)
    assert torch.equal(out, want_out) and torch.equal(state, ref)


def test_refusals(cuda):
    rec = pkg_module("recurrence")
    x = torch.zeros(4, 2, 8, device=cuda)
    bad = [
        (TypeError, lambda: rec.gated_scan(x.double(), x.double())),
        (TypeError, lambda: rec.gated_scan(x.half(), x)),
        (ValueError, lambda: rec.gated_scan(x[0], x[0])),
        (ValueError, lambda: rec.gated_scan(x[:2], x)),
        (ValueError, lambda: rec.gated_scan(x.cpu(), x.cpu())),
        (TypeError, lambda: rec.gated_scan(x, x, x[0].half())),
        (ValueError, lambda: rec.gated_scan(x, x, x[0, :1])),
        (TypeError, lambda: rec.gated_scan(x, x, reset=x[:, :, 0].long())),
        (ValueError, lambda: rec.gated_scan(x, x, reset=x[:, 0, 0])),
        (TypeError, lambda: rec.linear_scan(x, x, lengths=torch.ones(2, device=cuda, dtype=torch.int32))),
        (ValueError, lambda: rec.linear_scan(x, x, lengths=torch.ones(3, device=cuda, dtype=torch.int64))),
        (TypeError, lambda: rec.gated_step(x[0].half(), x[0].half(), x[0].half())),
        (ValueError, lambda: rec.gated_step(x[0], x[0], torch.zeros(2, 9, device=cuda))),
        (ValueError, lambda: rec.gated_step(x[0], x[0], torch.zeros(8, 2, device=cuda).t())),
        (ValueError, lambda: rec.gated_step(x[0], x[0], torch.zeros(1, 8, device=cuda).expand(2, 8))),
        (ValueError, lambda: rec.gated_step(x, x, x)),
        (ValueError, lambda: rec.linear_step(x[0], x[0], x[1], out=torch.zeros(8, 2, device=cuda).t())),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
