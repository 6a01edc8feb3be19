"""The training operators past 2^31 elements and bytes, on a B200: offsets are 64-bit.  Only the far ends are
compared, against the same operators on copies of them (which the operators' own tests compare with fp64)."""
import pytest
import torch

from conftest import pkg_module

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory(cuda):
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    yield
    torch.cuda.empty_cache()


def test_layer_norm_rows_past_32_bits(cuda):
    ln = pkg_module("layernorm")
    rows, dim = 300_000, 8000                          # 2.4e9 values
    x = torch.empty(rows, dim, device=cuda, dtype=torch.bfloat16)
    x[-64:].copy_(torch.randn(64, dim, device=cuda))
    x[:-64] = 1.0
    w = torch.randn(dim, device=cuda, requires_grad=True)
    xs = x.requires_grad_()
    y = ln.layer_norm(xs, w)
    end = x.detach()[-64:].clone().requires_grad_()
    ye = ln.layer_norm(end, w)
    assert torch.equal(y[-64:], ye) and bool((y[:4] == 0).all())
    dy = torch.zeros_like(x)
    dy[-64:] = torch.randn(64, dim, device=cuda)
    dx, dw = torch.autograd.grad(y, (xs, w), dy)
    dxe, dwe = torch.autograd.grad(ye, (end, w), dy[-64:])
    assert torch.equal(dx[-64:], dxe) and bool((dx[:4] == 0).all())
    # the rows lie in other blocks: sums of 64 terms in another order
    assert float((dw - dwe).abs().max()) <= 64 * 2.0 ** -24 * 64 * 16


def test_scan_strides_past_32_bits(cuda):
    """Steps 1.1e9 values apart: the far ones lie past 2^31 values."""
    rec = pkg_module("recurrence")
    big = torch.zeros(3, 1_100_000_000, device=cuda, dtype=torch.bfloat16)
    far = lambda at: big.view(3, -1)[:, at:at + 2 * 64].view(3, 2, 64)
    gate, x = far(0), far(1_000_000_000)
    gate.copy_(torch.randn(3, 2, 64, device=cuda))
    x.copy_(torch.randn(3, 2, 64, device=cuda))
    assert gate.stride(0) * 2 > 2 ** 31
    dh = torch.randn(3, 2, 64, device=cuda).bfloat16()
    out = []
    for g, v in ((gate, x), (gate.contiguous(), x.contiguous())):
        g, v = g.detach().requires_grad_(), v.detach().requires_grad_()
        h, hn = rec.gated_scan(g, v)
        out.append((h.detach(), hn.detach(), *torch.autograd.grad(h, (g, v), dh)))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    state = [torch.zeros(2, 64, device=cuda) for _ in range(2)]
    rows = big.view(-1).as_strided((2, 64), (2_200_000_000, 1))
    a = rec.gated_step(rows, rows, state[0])
    b = rec.gated_step(rows.contiguous(), rows.contiguous(), state[1])
    assert torch.equal(a, b) and torch.equal(*state)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_tensor_past_32_bits(cuda, bits):
    """A tensor of 2.2e9 values and a small one behind it, whose moments lie past 2^31 in the flat buffers."""
    optim = pkg_module("optim")
    n = 2_200_000_000 if bits == 8 else 2_150_000_000
    p = torch.zeros(n, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    p.grad = torch.zeros(n, device=cuda, dtype=torch.bfloat16)
    p.grad[-1000:] = torch.randn(1000, device=cuda)
    q = torch.randn(777, device=cuda).bfloat16().requires_grad_()
    q.grad = torch.randn(777, device=cuda).bfloat16()
    # the same far ends by themselves (a whole number of scale blocks before them)
    cut = (n - 1000) // 256 * 256
    ps, qs = p.detach()[cut:].clone().requires_grad_(), q.detach().clone().requires_grad_()
    ps.grad, qs.grad = p.grad[cut:].clone(), q.grad.clone()
    kw = dict(lr=1e-2, state_bits=bits, master_weights=False, max_grad_norm=0.25)
    big, small = optim.AdamW([p, q], **kw), optim.AdamW([ps, qs], **kw)
    big.step()
    small.step()
    assert bool((p[:4096] == 0).all())
    # the norm is the same sum over other blocks: equal but for fp64's rounding, so the clip is too
    assert torch.equal(big.grad_norm, small.grad_norm)
    assert torch.equal(p[cut:], ps) and torch.equal(q, qs)
    a, b = big.state[q], small.state[qs]
    if bits == 32:
        assert torch.equal(a["exp_avg"], b["exp_avg"]) and torch.equal(a["exp_avg_sq"], b["exp_avg_sq"])
    else:
        # the rounding goes by the position in the flat buffers: the scales agree, the codes by a step at most
        assert torch.equal(a["exp_avg_scale"], b["exp_avg_scale"])
        x, y = a["exp_avg"].float(), b["exp_avg"].float()
        assert float(((x - y).abs() / y.abs().clamp_min(2.0 ** -6)).max()) <= 0.126
