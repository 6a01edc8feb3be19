"""AdamW over many tensors a launch, the gradients' clip included, moments in 32 or 8 bits.

A step is one launch for each group's parameters of one type (up to 720 tensors each), and one more of each for
the gradients' norm where they are clipped.

``AdamW`` is ``torch.optim.AdamW`` (decoupled weight decay; with ``weight_decay=0`` torch.optim.Adam,
the reference's optimiser, R/cuda_fdm/ppo_gpu.py:1300) for CUDA parameters, as a
``torch.optim.Optimizer``: groups, schedulers, ``state_dict`` as usual.  What it adds:

* ``max_grad_norm`` scales the gradients as ``torch.nn.utils.clip_grad_norm_`` over all parameters
  does, without a pass that rewrites them; ``grad_norm`` is the norm of the last step, on the device.
* ``state_bits=8`` keeps exp_avg as e4m3 and exp_avg_sq as e5m2 with a fp32 scale for every 256
  values: 2 bytes a parameter in place of 8.  The codes are rounded stochastically (a hash of seed, step
  and position): a moment moves by far less than a code's step at a time, rounded to nearest it would
  stay where it is.
* ``master_weights`` (16-bit parameters): fp32 copies that are updated and rounded into the
  parameters, without which an update below half a step of the parameter is lost.  A parameter that was set
  from outside since (a loaded checkpoint) is taken as it is.
* Step counts live on the device: a step captured into a CUDA graph counts on every replay.  The
  learning rate and the other numbers are those of the capture.

Moments, masters and step counts of a group's tensors of one type lie in flat buffers
(``state_buffers``); ``state[p]`` holds the tensors' views of them.

What torch's has and this one refuses: a tensor as ``lr``, a state of ``torch.optim.AdamW`` (its keys and step
counts differ; ``load_state_dict`` takes this class's own form), copies and pickles of the optimiser,
sparse gradients, parameters that are not contiguous or lie on several devices, groups changed other than by
``add_param_group``.  ``amsgrad``, ``maximize``, ``foreach``, ``capturable`` and ``differentiable`` are not arguments.
"""
import ctypes as C
import operator

import torch

from . import _lib

BLOCK = 256                     # F16_ADAMW_BLOCK: values that share a scale
LAUNCH_TENSORS, LAUNCH_PARTIALS = 720, 592      # tensors of one launch, and the partial sums it may write


_grad, _nbytes, _dtype = (operator.attrgetter(name) for name in ("grad", "nbytes", "dtype"))
_numel, _device, _contiguous, _address = (torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous,
                                          torch.Tensor.data_ptr)


class _Bucket:
    """The tensors of one type in a parameter group, and their state in flat buffers."""

    def __init__(self, params, bits, master):
        self.params = params
        self.dtype, self.device = params[0].dtype, params[0].device
        self.firsts, total = [], 0
        for p in params:
            self.firsts.append(total)
            total += -(-p.numel() // BLOCK) * BLOCK
        zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=self.device)
        self.buffers = {}
        if bits == 8:
            self.buffers["exp_avg"] = zeros(total, torch.float8_e4m3fn)
            self.buffers["exp_avg_scale"] = zeros(total // BLOCK, torch.float32)
            self.buffers["exp_avg_sq"] = zeros(total, torch.float8_e5m2)
            self.buffers["exp_avg_sq_scale"] = zeros(total // BLOCK, torch.float32)
        else:
            self.buffers["exp_avg"] = zeros(total, torch.float32)
            self.buffers["exp_avg_sq"] = zeros(total, torch.float32)
        if master:
            self.buffers["master"] = zeros(total, torch.float32)
        self.buffers["step"] = zeros(len(params), torch.int64)
        self.ticket = zeros(1, torch.int32)
        self.prepare(bits)

    def views(self, i):
        """The state of tensor i: views of the flat buffers."""
        n, first = self.params[i].numel(), self.firsts[i]
        out = {}
        for name, flat in self.buffers.items():
            if name == "step":
                out[name] = flat[i]
            elif name.endswith("_scale"):
                out[name] = flat[first // BLOCK:first // BLOCK - (-n // BLOCK)]
            else:
                out[name] = flat[first:first + n].view(self.params[i].shape)
        return out

    def clear_tails(self):
        """Zero behind the tensors' ends: what a step expects there, and no tensor's state holds."""
        for p, first in zip(self.params, self.firsts):
            end = first + p.numel()
            if end % BLOCK:
                for name in ("exp_avg", "exp_avg_sq", "master"):
                    if name in self.buffers:
                        self.buffers[name][end:end + -end % BLOCK].zero_()

    def prepare(self, bits):
        """What every step's call has alike: the table of all tensors, and the flat buffers' addresses."""
        self.numels = [p.numel() for p in self.params]
        n = len(self.params)
        self.tables = ((C.c_void_p * n)(), (C.c_void_p * n)(), (C.c_int64 * n)(), (C.c_int64 * n)(), (C.c_int32 * n)())
        b = self.buffers
        at = lambda name: b[name].data_ptr() if name in b else None
        self.args = _lib.AdamwArgs(0, _lib.DTYPES[self.dtype], bits, *(C.addressof(t) for t in self.tables), 0, 0, 0, 0, 0,
                                   0, at("exp_avg"), at("exp_avg_sq"), at("exp_avg_scale"), at("exp_avg_sq_scale"),
                                   at("master"), at("step"), self.ticket.data_ptr())
        self.tabled = None          # the tensors that the last three tables hold

    def arguments(self):
        """(AdamwArgs whose tables hold the tensors with a gradient, these tensors, what has to stay alive until
        the launch), or None."""
        # maps over method descriptors: a step over hundreds of small tensors is bound by this loop
        params, numels, grads = self.params, self.numels, list(map(_grad, self.params))
        live = range(len(params))
        if type(None) in set(map(type, grads)) or 0 in numels:
            live = [i for i, g in enumerate(grads) if g is not None and numels[i]]
            if not live:
                return None
            params, grads, numels = [params[i] for i in live], [grads[i] for i in live], [numels[i] for i in live]
        # torch lets a gradient differ from its parameter only where the parameter's storage was swapped after
        # the gradient was set; sizes in bytes and devices are what a launch relies on
        size = self.dtype.itemsize
        if (list(map(_numel, params)) != numels or set(map(_dtype, params)) != {self.dtype}
                or list(map(_nbytes, grads)) != [size * n for n in numels]
                or set(map(_device, params + grads)) != {self.device.index} or not all(map(_contiguous, params))):
            raise RuntimeError("a parameter's or a gradient's size, type, device or layout is not what it was when the "
                               "optimiser was made (sparse gradients are not taken)")
        if not all(map(_contiguous, grads)):
            grads = [g.detach().contiguous() for g in grads]
        n = len(live)
        t = self.tables
        t[0][:n] = list(map(_address, params))
        t[1][:n] = list(map(_address, grads))
        if live != self.tabled:
            t[2][:n] = numels
            t[3][:n] = [self.firsts[i] for i in live]
            t[4][:n] = live
            self.tabled = live
        self.args.count = n
        return self.args, params, grads


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW on the sm_100a kernels (module docstring).

    state_bits       32 or 8, of exp_avg and exp_avg_sq
    max_grad_norm    limit of the gradients' norm over all groups, or None
    master_weights   fp32 copies of bf16 / fp16 parameters
    seed             of the 8-bit moments' rounding
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 max_grad_norm=None, master_weights=True, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError("max_grad_norm must be above 0, or None")
        self.state_bits, self.master_weights = int(state_bits), bool(master_weights)
        self.max_grad_norm, self.seed = max_grad_norm, int(seed) & (2 ** 64 - 1)
        self.grad_norm = None
        self._buckets = []          # one list of _Bucket for each group
        self._members = []          # its tensors
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @staticmethod
    def _check_numbers(group):
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            raise TypeError("lr must be a number")
        if not (lr >= 0.0 and group["eps"] >= 0.0 and group["weight_decay"] >= 0.0):
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError("betas must lie in [0, 1)")

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_numbers(group)
            kinds, seen = {}, set()
            for p in group["params"]:
                _lib.require_cuda_tensor(p, tuple(_lib.DTYPES), None, "AdamW parameter")
                if not p.is_contiguous():
                    raise ValueError("AdamW parameters must be contiguous")
                if id(p) in seen:
                    raise ValueError("a parameter appears twice in the group")
                seen.add(id(p))
                kinds.setdefault((p.dtype, p.device), []).append(p)
            if len({d for _, d in kinds} | {b.device for bs in self._buckets for b in bs}) > 1:
                raise ValueError("AdamW parameters must lie on one device")
            buckets = [_Bucket(ps, self.state_bits, self.master_weights and dtype != torch.float32)
                       for (dtype, _), ps in kinds.items()]
        except BaseException:
            self.param_groups.pop()
            raise
        self._buckets.append(buckets)
        self._members.append(list(group["params"]))
        for b in buckets:
            for i, p in enumerate(b.params):
                self.state[p] = b.views(i)

    def __getstate__(self):
        raise TypeError("AdamW is not copied or pickled; make a new one and load_state_dict into it")

    def state_buffers(self):
        """The flat buffers behind the state, one dict for each group and parameter type: "exp_avg",
        "exp_avg_sq" (with "_scale" each for 8-bit states), "master" where there are masters, "step".
        A tensor begins at a multiple of 256 values, in the order of the group's parameters."""
        return [b.buffers for bs in self._buckets for b in bs]

    def load_state_dict(self, state_dict):
        """Copies a state of the same form (state_bits, masters, shapes) into the flat buffers."""
        groups = state_dict["param_groups"]
        if len(groups) != len(self.param_groups) or any(
                len(g["params"]) != len(h["params"]) for g, h in zip(groups, self.param_groups)):
            raise ValueError("the state's parameter groups differ from the optimiser's")
        pairs = [(k, p) for g, h in zip(groups, self.param_groups) for k, p in zip(g["params"], h["params"])]
        for k, p in pairs:
            new, old = state_dict["state"].get(k), self.state[p]
            if new is not None and (new.keys() != old.keys() or any(
                    tuple(new[n].shape) != tuple(old[n].shape) or new[n].dtype != old[n].dtype for n in old)):
                raise ValueError("a tensor's state differs in form (state_bits, master_weights or shape)")
        for g, h in zip(groups, self.param_groups):
            self._check_numbers({**h, **{k: v for k, v in g.items() if k != "params"}})
        for g, h in zip(groups, self.param_groups):
            h.update({k: v for k, v in g.items() if k != "params"})
        for k, p in pairs:
            new = state_dict["state"].get(k)
            for n, t in self.state[p].items():
                t.zero_() if new is None else t.copy_(new[n])
        for b in [b for bs in self._buckets for b in bs]:
            b.clear_tails()

    def step(self, closure=None):
        """One step over every parameter with a gradient; returns the closure's loss, if any."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = []
        if len(self.param_groups) != len(self._members):
            raise RuntimeError("parameter groups are added with add_param_group, and not taken out")
        for group, members, buckets in zip(self.param_groups, self._members, self._buckets):
            self._check_numbers(group)
            params = group["params"]
            if len(params) != len(members) or not all(map(operator.is_, params, members)):
                raise RuntimeError("a group's parameters, or the groups' order, are not what they were when it was added")
            for b in buckets:
                made = b.arguments()
                if made is not None:
                    calls.append((group, b, *made))
        if not calls:
            return loss
        lib = _lib.load()
        device = calls[0][1].ticket
        with _lib.on_device(device):
            stream = _lib.raw_stream(device)
            partial, norm, used = None, None, 0
            if self.max_grad_norm is not None:
                room = sum([-(-a.count // LAUNCH_TENSORS) for _, _, a, _, _ in calls]) * LAUNCH_PARTIALS
                sums = torch.empty(room, dtype=torch.float64, device=device.device)
                partial = sums.data_ptr()
                self.grad_norm = torch.empty((), dtype=torch.float32, device=device.device)
                norm, n = self.grad_norm.data_ptr(), C.c_int(0)
                for _, _, a, _, _ in calls:
                    _lib.check(lib.f16_grad_squares(a.count, a.grads_host, a.numel_host, a.dtype, partial + 8 * used,
                                                    room - used, C.byref(n), stream), "f16_grad_squares")
                    used += n.value
            for group, _, a, params, _ in calls:
                a.lr, a.eps, a.weight_decay = group["lr"], group["eps"], group["weight_decay"]
                a.beta1, a.beta2 = group["betas"]
                a.max_norm, a.partial, a.partials, a.norm = self.max_grad_norm or 0.0, partial, used, norm
                a.seed = self.seed
                _lib.check(lib.f16_adamw_step(C.byref(a), stream), "f16_adamw_step")
                torch.autograd.graph.increment_version(params)      # written behind autograd's back
        return loss
