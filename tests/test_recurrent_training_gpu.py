"""The training operators together on a B200, as a recurrent actor-critic uses them: LayerNorm ->
split-product Linear -> gated_scan over a rollout with episode ends -> Linear heads, trained by AdamW;
and the same network deciding step by step.

Against the same network in fp64 (torch modules, the recurrence as a loop): outputs and every gradient
within 1e-5 of the largest (the split products' tolerance; the other operators add less), one AdamW
step's parameters within 1e-5 of lr of the formula's on the fp64 gradients where those are not small
(a gradient near zero divides by itself).  Step by step, states within 1e-5 of the sequence's.
"""
import pytest
import torch
import torch.nn as nn

from conftest import pkg_module

pytestmark = pytest.mark.gpu

OBS, DIM, T, N = 184, 128, 24, 96


class Core(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = pkg_module("layernorm").LayerNorm(OBS)
        self.into = nn.Linear(OBS, 2 * DIM)
        self.post = pkg_module("layernorm").LayerNorm(DIM)
        self.head = nn.Linear(DIM, 84)

    def gates(self, obs):
        sm = pkg_module("splitmm")
        z = sm.run_tower(nn.Sequential(self.norm, self.into), obs.reshape(-1, OBS))
        return z.view(*obs.shape[:-1], 2 * DIM).split(DIM, -1)

    def read(self, h):
        sm = pkg_module("splitmm")
        return sm.run_tower(nn.Sequential(self.post, self.head), h.reshape(-1, DIM)).view(*h.shape[:-1], 84)

    def forward(self, obs, h0, done):
        gate, x = self.gates(obs)
        h, hn = pkg_module("recurrence").gated_scan(gate, x, h0, reset=done)
        return self.read(h), hn


def plain(core, obs, h0, done):
    """The same in fp64 from torch's elementary operations, with leaves of its own."""
    p = {k: v.detach().double().requires_grad_() for k, v in core.named_parameters()}
    norm = lambda v, n: nn.functional.layer_norm(v, v.shape[-1:], p[n + ".weight"], p[n + ".bias"])
    gate, x = (norm(obs.double(), "norm") @ p["into.weight"].t() + p["into.bias"]).split(DIM, -1)
    f, h, hs = torch.sigmoid(gate), h0.double(), []
    for t in range(obs.shape[0]):
        h = f[t] * torch.where(done[t].bool().unsqueeze(1), torch.zeros_like(h), h) + (1 - f[t]) * x[t]
        hs.append(h)
    return norm(torch.stack(hs), "post") @ p["head.weight"].t() + p["head.bias"], h, p


def case(cuda):
    torch.manual_seed(3)
    core = Core().to(cuda)
    g = torch.Generator(device=cuda).manual_seed(4)
    obs = torch.randn(T, N, OBS, device=cuda, generator=g)
    done = (torch.rand(T, N, device=cuda, generator=g) < 0.1).float()           # as PPOTrainer.b_done
    return core, obs, torch.randn(N, DIM, device=cuda, generator=g), done, torch.randn(T, N, 84, device=cuda, generator=g)


def rel(a, b):
    return float((a.double() - b).abs().max() / b.abs().max())


def test_training_step(cuda):
    core, obs, h0, done, dz = case(cuda)
    z, hn = core(obs, h0, done)
    ref_z, ref_hn, p = plain(core, obs, h0, done)
    assert rel(z.detach(), ref_z.detach()) <= 1e-5 and rel(hn.detach(), ref_hn.detach()) <= 1e-5
    z.backward(dz)
    grads = torch.autograd.grad(ref_z, list(p.values()), dz.double())
    for (name, q), g in zip(core.named_parameters(), grads):
        assert rel(q.grad, g) <= 1e-5, name
    lr, eps = 1e-3, 1e-5
    before = {k: v.detach().double() for k, v in core.named_parameters()}
    norm = torch.sqrt(sum((g ** 2).sum() for g in grads))
    c = min(1.0, 0.5 / (float(norm) + 1e-6))
    opt = pkg_module("optim").AdamW(core.parameters(), lr=lr, eps=eps, weight_decay=0.01, max_grad_norm=0.5)
    opt.step()
    assert abs(float(opt.grad_norm) - float(norm)) <= 1e-5 * float(norm)
    for (name, q), g in zip(core.named_parameters(), grads):
        want = before[name] * (1 - lr * 0.01) - lr * c * g / ((c * g).abs() + eps)
        sure = g.abs() > 1e-2 * g.abs().max()
        # d/dg of g/(|g| + eps) is at most 1/(|g| + eps): 1e-5 of the largest over 1e-2 of it
        assert float(((q.detach().double() - want).abs() * sure).max()) <= lr * 1e-3 + 2e-7, name


def test_decisions_equal_the_sequence(cuda):
    core, obs, h0, done, _ = case(cuda)
    rec = pkg_module("recurrence")
    with torch.no_grad():
        z, hn = core(obs, h0, done)
        state = h0.clone()
        for t in range(T):
            gate, x = core.gates(obs[t])
            out = core.read(rec.gated_step(gate, x, state, reset=done[t]))
            assert rel(out, z[t].double()) <= 1e-5
    assert rel(state, hn.double()) <= 1e-5


def test_many_steps_captured(cuda):
    """Forward, backward and AdamW (8-bit moments) captured once and replayed: the same parameters as the eager
    loop's, bit for bit.  Gradients are taken with torch.autograd.grad into fixed buffers: a captured
    backward() must not share its leaves' accumulators with an eager graph that is still alive."""
    optim = pkg_module("optim")
    results = []
    for captured in (False, True):
        core, obs, h0, done, dz = case(cuda)
        params = list(core.parameters())
        for p in params:
            p.grad = torch.zeros_like(p)
        opt = optim.AdamW(params, lr=1e-3, state_bits=8, max_grad_norm=1.0)

        def step():
            z, _ = core(obs, h0, done)
            for p, g in zip(params, torch.autograd.grad(z, params, dz)):
                p.grad.copy_(g)
            opt.step()

        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            for _ in range(3):
                graph.replay()
        else:
            for _ in range(4):
                step()
        torch.cuda.synchronize()
        results.append([p.detach().clone() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(*results))
