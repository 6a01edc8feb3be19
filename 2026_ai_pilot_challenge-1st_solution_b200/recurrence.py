"""A gated linear recurrence over time on the sm_100a kernels, with its gradient and its single step.

    linear_scan:  h_t = a_t h_{t-1} + x_t
    gated_scan:   f = sigmoid(gate_t),  h_t = f h_{t-1} + (1 - f) x_t

for each of batch x dim channels by itself, over time-major tensors (steps, batch, dim) as the
rollout buffers are (a batch-first tensor goes in as ``t.transpose(0, 1)``, a view).  ``reset[t, b]``
drops the state before step t (``PPOTrainer.b_done`` as it is: the step begins a new episode),
``lengths[b]`` ends a padded sequence: later steps leave the state, return zeros and get zero gradients,
and what they hold is not read.  The state is fp32 throughout; outputs have the inputs' type.

``gated_step`` / ``linear_step`` are one step of it for a decision, the fp32 state updated in place.

``rollout.gae`` is the recurrence of this kind that the framework had (in reverse time, with scalar
coefficients); the reference has no recurrent network left (its GRU was removed).
"""
import ctypes as C

import torch

from . import _lib

CHUNK = 16          # F16_SCAN_CHUNK: steps between the states that the forward pass saves


def _strided(t):
    """t with unit stride along dim (itself where it has it)."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _like(x):
    """An uninitialised tensor of x's shape in x's order of axes, without gaps."""
    out = torch.empty_like(x)
    return out if out.stride(2) == 1 or x.shape[2] == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _fill(args, name, t):
    setattr(args, name, t.data_ptr())
    setattr(args, name + "_t", t.stride(0))
    setattr(args, name + "_b", t.stride(1))


def _args(gate, x, h0, reset, lengths, gated):
    a = _lib.ScanArgs()
    a.dtype, a.gated = _lib.DTYPES[x.dtype], int(gated)
    a.steps, a.batch, a.dim = x.shape
    _fill(a, "gate", gate)
    _fill(a, "x", x)
    if h0 is not None:
        a.h0 = h0.data_ptr()
    if reset is not None:
        a.reset, a.reset_bytes = reset.data_ptr(), reset.element_size()
        a.reset_t, a.reset_b = reset.stride(0), reset.stride(1)
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    return a


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, reset, lengths, gated):
        ctx.set_materialize_grads(False)
        steps, batch, dim = x.shape
        gate, x = _strided(gate), _strided(x)
        h = _like(x)
        hn = torch.empty(batch, dim, dtype=torch.float32, device=x.device)
        if h0 is not None:
            h0 = h0.contiguous()
        saved = None
        if x.numel() == 0:
            hn.zero_() if h0 is None else hn.copy_(h0)
        else:
            lib = _lib.load()
            a = _args(gate, x, h0, reset, lengths, gated)
            _fill(a, "h", h)
            a.hn = hn.data_ptr()
            if any(ctx.needs_input_grad[:3]):
                saved = torch.empty(lib.f16_scan_saved_floats(steps, batch, dim), dtype=torch.float32, device=x.device)
                a.saved = saved.data_ptr()
            with _lib.on_device(x):
                _lib.check(lib.f16_scan_fwd(C.byref(a), _lib.stream_of(x)), "f16_scan_fwd")
        ctx.gated = gated
        ctx.save_for_backward(gate, x, h0, reset, lengths, saved)
        return h, hn

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dhn):
        gate, x, h0, reset, lengths, saved = ctx.saved_tensors
        if dh is None and dhn is None:
            return None, None, None, None, None, None
        need_gate, need_x, need_h0 = ctx.needs_input_grad[:3]
        batch, dim = x.shape[1:]
        dgate = _like(gate) if need_gate else None
        dx = _like(x) if need_x else None
        dh0 = torch.empty(batch, dim, dtype=torch.float32, device=x.device) if need_h0 else None
        if x.numel() == 0:
            if dh0 is not None:
                dh0.zero_() if dhn is None else dh0.copy_(dhn)
            return dgate, dx, dh0, None, None, None
        a = _args(gate, x, h0, reset, lengths, ctx.gated)
        a.saved = saved.data_ptr()
        if dh is not None:
            dh = _strided(dh)
            _fill(a, "dh", dh)
        if dhn is not None:
            dhn = dhn.contiguous()
            a.dhn = dhn.data_ptr()
        if dgate is not None:
            _fill(a, "dgate", dgate)
        if dx is not None:
            _fill(a, "dx", dx)
        if dh0 is not None:
            a.dh0 = dh0.data_ptr()
        with _lib.on_device(x):
            _lib.check(_lib.load().f16_scan_bwd(C.byref(a), _lib.stream_of(x)), "f16_scan_bwd")
        return dgate, dx, dh0, None, None, None


def _flags(reset, shape, device):
    _lib.require_cuda_tensor(reset, (torch.bool, torch.uint8, torch.float32), shape, "reset flags", device)
    return reset


def _scan(gate, x, h0, reset, lengths, gated, name):
    _lib.require_cuda_tensor(x, tuple(_lib.DTYPES), None, f"{name} input")
    if x.dim() != 3:
        raise ValueError(f"{name} takes (steps, batch, dim) tensors")
    _lib.require_cuda_tensor(gate, x.dtype, x.shape, "gate" if gated else "coefficients", x.device)
    steps, batch, dim = x.shape
    if h0 is not None:
        _lib.require_cuda_tensor(h0, torch.float32, (batch, dim), "initial state", x.device)
    if reset is not None:
        _flags(reset, (steps, batch), x.device)
    if lengths is not None:
        _lib.require_cuda_tensor(lengths, torch.int64, (batch,), "lengths", x.device)
        lengths = lengths.contiguous()
    return _Scan.apply(gate, x, h0, reset, lengths, gated)


def gated_scan(gate, x, h0=None, reset=None, lengths=None):
    """(h, hn) of h_t = f h_{t-1} + (1 - f) x_t, f = sigmoid(gate_t), from h0 (zero where None).

    gate, x     (steps, batch, dim) fp32, bf16 or fp16, the same type; any strides along time and batch
    h0          (batch, dim) fp32
    reset       (steps, batch) bool, uint8 or fp32 flags
    lengths     (batch,) int64, taken as at least 0 and at most steps
    h           the states in the inputs' type; hn: the last one, (batch, dim) fp32
    """
    return _scan(gate, x, h0, reset, lengths, True, "gated_scan")


def linear_scan(a, x, h0=None, reset=None, lengths=None):
    """(h, hn) of h_t = a_t h_{t-1} + x_t; arguments as in ``gated_scan``.  Meant for coefficients of
    size up to 1; the product of 256 successive ones has to stay in fp32's range."""
    return _scan(a, x, h0, reset, lengths, False, "linear_scan")


@torch.no_grad()
def _step(gate, x, state, reset, out, gated, name):
    _lib.require_cuda_tensor(x, tuple(_lib.DTYPES), None, f"{name} input")
    if x.dim() != 2:
        raise ValueError(f"{name} takes (batch, dim) tensors")
    _lib.require_cuda_tensor(gate, x.dtype, x.shape, "gate" if gated else "coefficients", x.device)
    _lib.require_cuda_tensor(state, torch.float32, x.shape, "state", x.device)
    batch, dim = x.shape
    if out is None:
        out = torch.empty(batch, dim, dtype=x.dtype, device=x.device)
    else:
        _lib.require_cuda_tensor(out, x.dtype, x.shape, "output", x.device)
    for t, label in ((state, "state"), (out, "output")):
        if batch and dim and (dim > 1 and t.stride(1) != 1 or batch > 1 and t.stride(0) < dim):
            raise ValueError(f"{label} rows must be contiguous and apart")
    if reset is not None:
        _flags(reset, (batch,), x.device)
    if x.numel() == 0:
        return out
    if dim > 1:
        gate = gate if gate.stride(1) == 1 else gate.contiguous()
        x = x if x.stride(1) == 1 else x.contiguous()
    rows = lambda t: t.stride(0) if batch > 1 else dim
    with _lib.on_device(x):
        _lib.check(_lib.load().f16_scan_step(
            gate.data_ptr(), rows(gate), x.data_ptr(), rows(x), batch, dim, _lib.DTYPES[x.dtype], int(gated),
            _lib.ptr(reset), reset.element_size() if reset is not None else 0,
            reset.stride(0) if reset is not None else 0, state.data_ptr(), rows(state), out.data_ptr(), rows(out),
            _lib.stream_of(x)), "f16_scan_step")
    torch.autograd.graph.increment_version((state, out))
    return out


def gated_step(gate, x, state, reset=None, out=None):
    """One step of ``gated_scan`` for a decision: gate, x (batch, dim), state (batch, dim) fp32 updated in
    place, reset (batch,) flags or None.  Returns the new state in the inputs' type (``out``); no
    gradient is recorded."""
    return _step(gate, x, state, reset, out, True, "gated_step")


def linear_step(a, x, state, reset=None, out=None):
    """One step of ``linear_scan``; arguments as in ``gated_step``."""
    return _step(a, x, state, reset, out, False, "linear_step")
