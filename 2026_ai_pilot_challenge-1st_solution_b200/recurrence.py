"""A gated linear recurrence over time on the sm_100a kernels, with its gradient and its single step.

    linear_scan:  h_t = a_t h_{t-1} + x_t
    gated_scan:   f = sigmoid(gate_t),  h_t = f h_{t-1} + (1 - f) x_t

for each of batch x dim channels by itself, over time-major tensors (steps, batch, dim) as the
rollout buffers are (a batch-first tensor goes in as ``t.transpose(0, 1)``, a view).  ``reset[t, b]``
drops the state before step t (``PPOTrainer.b_done`` as it is: the step begins a new episode),
``lengths[b]`` ends a padded sequence: later steps leave the state, return zeros and get zero gradients,
and what they hold is not read.  The state is fp32 throughout; outputs have the inputs' type.
Forward-mode derivatives, double backward and functorch transforms are refused.

A state that becomes infinite or NaN stays one of the two until a reset, as does an infinite gradient until the
reset before it; which of the two can depend on how the call is cut into segments (where coefficients
multiply to 0 before they meet an infinite state).

``gated_step`` / ``linear_step`` are one step of it for a decision, the fp32 state updated in place.  They are for
a loop of the user's own: ``PPOTrainer``'s policies have no state, and ``ppo_update`` draws rows without regard to time.

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


_FLOATS, _FLAGS, _F32, _I64 = tuple(_lib.DTYPES), (torch.bool, torch.uint8, torch.float32), (torch.float32,), (torch.int64,)


def _place(t):
    """(address, time stride, batch stride) of a sequence tensor or None."""
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


def _at(t):
    return None if t is None else t.data_ptr()


def _scratch(lib, x):
    """(buffer, values in it) for the segments of a scan with few channels, or (None, 0)."""
    n = lib.f16_scan_scratch_floats(*map(int, x.shape))      # a trace has tensors there
    return (x.new_empty(n, dtype=torch.float32) if n else None), n


def _args(gate, x, h0, reset, lengths, gated, h, hn, saved, scratch, dh=None, dhn=None, dgate=None, dx=None, dh0=None):
    return _lib.ScanArgs(_lib.DTYPES[x.dtype], gated, *map(int, x.shape), *_place(gate), *_place(x), _at(h0), _at(reset),
                         reset.element_size() if reset is not None else 0,
                         *(reset.stride() if reset is not None else (0, 0)), _at(lengths), *_place(h), _at(hn), _at(saved),
                         *_place(dh), _at(dhn), *_place(dgate), *_place(dx), _at(dh0),
                         _at(scratch[0]), scratch[1])


def _forward(gate, x, h0, reset, lengths, gated, keep):
    """(h, hn, the states that the backward pass needs if ``keep``); gate and x with unit stride along dim."""
    steps, batch, dim = map(int, x.shape)
    h = _like(x)
    hn = x.new_empty(batch, dim, dtype=torch.float32)
    saved = None
    if not x.numel():
        hn.zero_() if h0 is None else hn.copy_(h0)
    else:
        lib = _lib.load()
        if keep:
            saved = x.new_empty(lib.f16_scan_saved_floats(steps, batch, dim), dtype=torch.float32)
        with _lib.on_device(x):
            scratch = _scratch(lib, x)
            a = _args(gate, x, h0, reset, lengths, gated, h, hn, saved, scratch)
            _lib.check(lib.f16_scan_fwd(C.byref(a), _lib.raw_stream(x)), "f16_scan_fwd")
    return h, hn, saved


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, reset, lengths, gated):
        ctx.set_materialize_grads(False)
        gate, x = _strided(gate), _strided(x)
        h, hn, saved = _forward(gate, x, h0, reset, lengths, gated, True)
        ctx.gated = gated
        ctx.save_for_backward(gate, x, h0, reset, lengths, saved)
        return h, hn

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dhn):
        if dh is None and dhn is None:
            return None, None, None, None, None, None
        gate, x, h0, reset, lengths, saved = ctx.saved_tensors
        need_gate, need_x, need_h0 = ctx.needs_input_grad[:3]
        dgate = _like(gate) if need_gate else None
        dx = _like(x) if need_x else None
        dh0 = x.new_empty(x.shape[1:], dtype=torch.float32) if need_h0 else None
        if not x.numel():
            if dh0 is not None:
                dh0.zero_() if dhn is None else dh0.copy_(dhn)
            return dgate, dx, dh0, None, None, None
        dh = _strided(dh) if dh is not None else None
        dhn = dhn.contiguous() if dhn is not None else None
        lib = _lib.load()
        with _lib.on_device(x):
            scratch = _scratch(lib, x)
            a = _args(gate, x, h0, reset, lengths, ctx.gated, None, None, saved, scratch, dh, dhn, dgate, dx, dh0)
            _lib.check(lib.f16_scan_bwd(C.byref(a), _lib.raw_stream(x)), "f16_scan_bwd")
        return dgate, dx, dh0, None, None, None


def _scan(gate, x, h0, reset, lengths, gated, name):
    _lib.checked(x, _FLOATS, None, f"{name} input")
    if x.dim() != 3:
        raise ValueError(f"{name} takes (steps, batch, dim) tensors")
    _lib.checked(gate, (x.dtype,), x.shape, "gate" if gated else "coefficients", x)
    if h0 is not None:
        h0 = _lib.checked(h0, _F32, x.shape[1:], "initial state", x).contiguous()
    if reset is not None:
        _lib.checked(reset, _FLAGS, x.shape[:2], "reset flags", x)
    if lengths is not None:
        lengths = _lib.checked(lengths, _I64, x.shape[1:2], "lengths", x).contiguous()
    if _lib.transformed(gate, x, h0) or torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or h0 is not None and h0.requires_grad):
        return _Scan.apply(gate, x, h0, reset, lengths, int(gated))
    return _forward(_strided(gate), _strided(x), h0, reset, lengths, int(gated), False)[:2]


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
    size up to 1.  Where larger ones are among them, the product of any up to 8,192 successive ones has to stay
    in fp32's normal range: a call with few channels multiplies them before they meet the state, where one
    with many does not."""
    return _scan(a, x, h0, reset, lengths, False, "linear_scan")


def _step(gate, x, state, reset, out, gated, name):
    _lib.checked(x, _FLOATS, None, f"{name} input")
    if x.dim() != 2:
        raise ValueError(f"{name} takes (batch, dim) tensors")
    shape = x.shape
    _lib.checked(gate, (x.dtype,), shape, "gate" if gated else "coefficients", x)
    _lib.checked(state, _F32, shape, "state", x)
    if out is None:
        out = x.new_empty(shape)
    else:
        _lib.checked(out, (x.dtype,), shape, "output", x)
    if reset is not None:
        _lib.checked(reset, _FLAGS, shape[:1], "reset flags", x)
    _lib.refuse_transformed(name, gate, x, state, out)
    batch, dim = shape
    if not batch or not dim:
        return out
    for t, label in ((state, "state"), (out, "output")):
        if not t.is_contiguous() and (dim > 1 and t.stride(1) != 1 or batch > 1 and t.stride(0) < dim):
            raise ValueError(f"{label} rows must be contiguous and apart")
    if dim > 1:
        gate = gate if gate.stride(1) == 1 else gate.contiguous()
        x = x if x.stride(1) == 1 else x.contiguous()
    rows = [t.stride(0) if batch > 1 else dim for t in (gate, x, state, out)]
    with _lib.on_device(x):
        _lib.check(_lib.load().f16_scan_step(
            gate.data_ptr(), rows[0], x.data_ptr(), rows[1], batch, dim, _lib.DTYPES[x.dtype], gated, _at(reset),
            reset.element_size() if reset is not None else 0, reset.stride(0) if reset is not None else 0,
            state.data_ptr(), rows[2], out.data_ptr(), rows[3], _lib.raw_stream(x)), "f16_scan_step")
    torch.autograd.graph.increment_version((state, out))      # written behind autograd's back
    return out


def gated_step(gate, x, state, reset=None, out=None):
    """One step of ``gated_scan`` for a decision: gate, x (batch, dim), state (batch, dim) fp32 updated in
    place, reset (batch,) flags or None.  Returns the new state in the inputs' type (``out``); no
    gradient is recorded, traces and transforms are refused.
    ``out`` and ``state`` may be x's or gate's own memory, but share no part of it at another place."""
    return _step(gate, x, state, reset, out, 1, "gated_step")


def linear_step(a, x, state, reset=None, out=None):
    """One step of ``linear_scan``; arguments as in ``gated_step``."""
    return _step(a, x, state, reset, out, 0, "linear_step")
