"""Layer norm over the last axis on the sm_100a kernels, with its gradient.

``layer_norm(x, weight, bias, eps)`` is ``torch.nn.functional.layer_norm`` over the last axis for CUDA
tensors: fp32, bf16 or fp16 input, weight and bias in fp32 or the input's type (either may be
None), statistics and sums in fp32, one rounding when a value is stored.  Under ``torch.autocast`` 16-bit
arguments are taken as fp32 and so is the output, as torch's.  fp64 inputs are refused.  Backward gives the
gradients of x, weight and bias in two launches (three for rows too wide for registers); the sums over rows
behind the weight's and bias's are made in a fixed order, so the same inputs give the same bits.  Forward-mode derivatives, double backward
and functorch transforms are refused.  ``LayerNorm`` is
``torch.nn.LayerNorm`` over one axis with that forward (CPU tensors take torch's): it
keeps the parameter names, and ``splitmm.run_tower`` takes it between its layers.  ``trainer.MLPActorCritic`` builds no
towers with it, and ``policy.MlpWeights`` (the rollout's fused forward) refuses one.

The reference normalises observations only (``rollout.RunningNorm``) and has no counterpart.
"""
import torch

from . import _lib


_FLOATS = tuple(_lib.DTYPES)
_HALVES = (torch.bfloat16, torch.float16)
MAX_DIM = 2 ** 29


def _rows(x):
    """x as (rows, dim) with unit column stride (a view where its layout allows)."""
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    return x if x.stride(1) == 1 and x.stride(0) >= 0 or x.shape[1] == 1 else x.contiguous()


def _row_stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _forward(x, rows, weight, bias, eps, stats):
    n, dim = map(int, rows.shape)           # a trace has tensors there
    y = x.new_empty(x.shape)
    if n:
        wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
        at = stats.data_ptr() if stats is not None else None
        with _lib.on_device(x):
            _lib.check(_lib.load().f16_layer_norm_fwd_rest(
                rows.data_ptr(), n, dim, _row_stride(rows), _lib.DTYPES[x.dtype],
                weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None,
                _lib.DTYPES[wdtype], eps, y.data_ptr(), dim, at, at + 4 * n if at is not None else None,
                at + 8 * n if at is not None else None, _lib.raw_stream(x)), "f16_layer_norm_fwd")
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = _rows(x)
        stats = x.new_empty(3, rows.shape[0], dtype=torch.float32)      # mean, what its rounding left, 1 / deviation
        ctx.wdtype = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
        ctx.save_for_backward(rows, weight, stats)
        return _forward(x, rows, weight, bias, eps, stats)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        n, dim = x.shape
        shape = dy.shape
        dy = _rows(dy)
        dx = x.new_empty(shape) if need_x else None
        if not n:
            zero = torch.zeros(dim, dtype=ctx.wdtype, device=x.device) if need_w or need_b else None
            return dx, zero if need_w else None, zero.clone() if need_b else None, None
        dw = x.new_empty(dim, dtype=ctx.wdtype) if need_w else None
        db = x.new_empty(dim, dtype=ctx.wdtype) if need_b else None
        lib = _lib.load()
        with _lib.on_device(x):
            room = lib.f16_layer_norm_scratch_floats(n, dim) if need_w or need_b else 0
            scratch = x.new_empty(room, dtype=torch.float32) if room else None
            at = stats.data_ptr()
            _lib.check(lib.f16_layer_norm_bwd_rest(
                dy.data_ptr(), _row_stride(dy), x.data_ptr(), _row_stride(x), n, dim, _lib.DTYPES[x.dtype],
                weight.data_ptr() if weight is not None else None, _lib.DTYPES[ctx.wdtype], at, at + 4 * n, at + 8 * n,
                dx.data_ptr() if need_x else None, dim, dw.data_ptr() if need_w else None,
                db.data_ptr() if need_b else None, scratch.data_ptr() if room else None, room,
                _lib.raw_stream(x)), "f16_layer_norm_bwd")
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (module docstring)."""
    if torch.is_autocast_enabled("cuda"):
        x, weight, bias = (t.float() if torch.is_tensor(t) and t.dtype in _HALVES else t for t in (x, weight, bias))
    _lib.checked(x, _FLOATS, None, "layer_norm input")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError("layer_norm needs a last axis of 1 to 2^29 values")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    shape = x.shape[-1:]
    if weight is not None:
        weight = _lib.checked(weight, (torch.float32, x.dtype), shape, "layer_norm weight", x).contiguous()
    if bias is not None:
        bias = _lib.checked(bias, (torch.float32, x.dtype), shape, "layer_norm bias", x).contiguous()
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError("layer_norm weight and bias must have the same dtype")
    if _lib.transformed(x, weight, bias) or torch.is_grad_enabled() and (
            x.requires_grad or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, _rows(x), weight, bias, float(eps), None)


class LayerNorm(torch.nn.LayerNorm):
    """torch.nn.LayerNorm over the last axis; CUDA tensors run through ``layer_norm``."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises the last axis only")

    def forward(self, x):
        if not x.is_cuda:
            return super().forward(x)
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"input's last axis {tuple(x.shape[-1:])} != {tuple(self.normalized_shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
