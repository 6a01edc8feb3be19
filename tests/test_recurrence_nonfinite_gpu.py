"""A state that becomes infinite or NaN in recurrence.gated_scan, on a B200, with time cut into segments and not:
the same elements are finite, whatever number stands in the others, and those that are agree."""
import ctypes

import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu


def run(d, scratch, gated):
    _lib, rec = pkg_module("_lib"), pkg_module("recurrence")
    lib = _lib.load()
    steps, batch, dim = d["x"].shape
    new = lambda *s: torch.empty(*s, device=d["x"].device)
    saved = new(lib.f16_scan_saved_floats(steps, batch, dim))
    out = dict(h=torch.empty_like(d["x"]), hn=new(batch, dim), dgate=torch.empty_like(d["x"]), dx=torch.empty_like(d["x"]),
               dh0=new(batch, dim))
    s = (scratch, 0 if scratch is None else scratch.numel())
    a = rec._args(d["gate"], d["x"], d["h0"], d["reset"], None, gated, out["h"], out["hn"], saved, s)
    _lib.check(lib.f16_scan_fwd(ctypes.byref(a), _lib.stream_of(d["x"])), "f16_scan_fwd")
    a = rec._args(d["gate"], d["x"], d["h0"], d["reset"], None, gated, None, None, saved, s, d["dh"], d["dhn"],
                  out["dgate"], out["dx"], out["dh0"])
    _lib.check(lib.f16_scan_bwd(ctypes.byref(a), _lib.stream_of(d["x"])), "f16_scan_bwd")
    return out


@pytest.mark.parametrize("gated", [1, 0])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_the_same_elements_are_finite(cuda, gated, value):
    """4,096 steps; channel 1 is given the value at step 700 and dropped at step 3,000, channel 2's gradient at step
    2,500.  Coefficients of 0.3 to 0.6: a segment's product underflows.  The others agree within the roundings
    of a decay of 0.6 (32 half steps a step in each of two runs, over 1 / 0.4), of values of at most 16."""
    g = torch.Generator(device=cuda).manual_seed(4)
    rnd = lambda *s: torch.randn(*s, device=cuda, generator=g)
    steps = 4096
    a = 0.3 + 0.3 * torch.rand(steps, 1, 40, device=cuda, generator=g)
    d = dict(gate=torch.logit(a) if gated else a, x=rnd(steps, 1, 40), h0=rnd(1, 40), dh=rnd(steps, 1, 40), dhn=rnd(1, 40),
             reset=torch.zeros(steps, 1, device=cuda, dtype=torch.bool))
    d["reset"][3000] = True
    d["x"][700, 0, 1] = value
    d["dh"][2500, 0, 2] = value
    n = pkg_module("_lib").load().f16_scan_scratch_floats(steps, 1, 40)
    assert n > 0
    cut, uncut = run(d, torch.empty(n, device=cuda), gated), run(d, None, gated)
    bad = torch.zeros(steps, 40, dtype=torch.bool, device=cuda)
    bad[700:3000, 1] = True
    assert torch.equal(cut["h"][:, 0].isfinite(), ~bad)
    bad = torch.zeros(steps, 40, dtype=torch.bool, device=cuda)
    bad[:2501, 2] = True
    assert torch.equal(cut["dx"][:, 0].isfinite(), ~bad)
    assert bool(cut["hn"].isfinite().all()) and cut["dh0"].isfinite().tolist() == [[i != 2 for i in range(40)]]
    for name in cut:
        fine = uncut[name].isfinite()
        assert torch.equal(cut[name].isfinite(), fine), name
        assert bool(((cut[name] - uncut[name])[fine].abs() <= 2 * 32 * 2.0 ** -24 / 0.4 * 16).all()), name
