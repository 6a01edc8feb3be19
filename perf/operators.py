"""Cases for the training operators: layer norm, the gated linear recurrence and the AdamW step.

``run`` computes one pass through an operator: with ``own`` false from elementary torch
operations, with ``own`` true through the package's public entry points (``layernorm.layer_norm``,
``recurrence.gated_scan`` / ``linear_scan`` / ``gated_step`` / ``linear_step``, ``optim.AdamW``).

A case is a dict of plain values; ``op`` names the operator:

  "norm"   rows x dim, dtype, wdtype (weight and bias: "float32" or the input's, "none": without
           them), train (with the gradients of input, weight and bias)
  "scan"   steps x batch x dim, dtype, gated (sigmoid gate) or raw coefficients, resets, padded
           (a length per sequence, some of them zero), initial (a state to begin with),
           batch_first (the tensors are transposed views of (batch, steps, dim) storage), train
  "step"   one time step over batch x dim, the fp32 state updated in place
  "adamw"  the tensors of `towers` networks of Linear layers, dim -> hidden (x layers) -> out;
           dtype, bits (of the moments), master (fp32 copies of 16-bit parameters), clip
           (the limit of the gradients' norm, 0: none)
"""
import math

import torch

own = False

PACKAGE = "2026_ai_pilot_challenge-1st_solution_b200"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 3e-4, 0.9, 0.999, 1e-5, 1e-2
STEPS_DONE = 100           # optimiser steps behind the state that prepare() makes
SEED = 1234                # of the 8-bit moments' rounding
BLOCK = 256                # moments that share a scale; tensors begin at multiples of it
RESET_RATE = 0.005         # episode ends per step


def _package(name):
    import importlib
    return importlib.import_module(PACKAGE + "." + name)


# ---------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decision of a small evaluation batch: observation rows before a policy
        {"name": "norm decision", "op": "norm", "rows": 128, "dim": 184, "dtype": "float32", "wdtype": "float32",
         "train": False},
        # one minibatch of the PPO update (131,072 environments x 64 decisions in 16 minibatches)
        # through the norm of a 512-wide hidden layer
        {"name": "norm minibatch", "op": "norm", "rows": 524288, "dim": 512, "dtype": "float32", "wdtype": "float32",
         "train": True},
        # a wide 16-bit trunk
        {"name": "norm wide", "op": "norm", "rows": 16384, "dim": 4096, "dtype": "bfloat16", "wdtype": "float32",
         "train": True},
        # the 214 external observation columns plus one, in fp16: rows off every alignment
        {"name": "norm odd", "op": "norm", "rows": 100003, "dim": 215, "dtype": "float16", "wdtype": "float16",
         "train": True},
        # a rollout of 64 decisions through a 128-wide recurrent core, episodes ending inside
        {"name": "scan rollout", "op": "scan", "steps": 64, "batch": 16384, "dim": 128, "dtype": "bfloat16",
         "gated": True, "resets": True, "padded": False, "initial": True, "batch_first": False, "train": True},
        # one long sequence: few channels, the work lies along time
        {"name": "scan long", "op": "scan", "steps": 65536, "batch": 1, "dim": 1024, "dtype": "bfloat16",
         "gated": True, "resets": False, "padded": False, "initial": False, "batch_first": False, "train": True},
        # recorded games of different lengths, padded, batch first, an odd width, raw coefficients
        {"name": "scan padded", "op": "scan", "steps": 1000, "batch": 37, "dim": 185, "dtype": "float32",
         "gated": False, "resets": True, "padded": True, "initial": True, "batch_first": True, "train": True},
        # one decision of an evaluation's environments through the core
        {"name": "step decision", "op": "step", "batch": 256, "dim": 512, "dtype": "bfloat16", "gated": True,
         "resets": True},
        # one decision of a training rollout's environments
        {"name": "step rollout", "op": "step", "batch": 131072, "dim": 128, "dtype": "float32", "gated": True,
         "resets": True},
        # actor and critic of the PPO update, its clip: sixteen small tensors
        {"name": "adamw policy", "op": "adamw", "towers": 2, "dim": 184, "hidden": 512, "layers": 3, "out": 84,
         "dtype": "float32", "bits": 32, "master": False, "clip": 0.5},
        # a large trunk in fp32 with 8-bit moments
        {"name": "adamw large 8 bit", "op": "adamw", "towers": 1, "dim": 4096, "hidden": 4096, "layers": 14,
         "out": 4096, "dtype": "float32", "bits": 8, "master": False, "clip": 1.0},
        # three hundred tensors of odd sizes in bf16, fp32 moments and master copies
        {"name": "adamw odd bf16", "op": "adamw", "towers": 1, "dim": 215, "hidden": 385, "layers": 149, "out": 85,
         "dtype": "bfloat16", "bits": 32, "master": True, "clip": 1.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "scan", "scan", "step", "adamw", "adamw"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "norm":
        dim = _log(rng, 1, 20000)
        if rng.random() < 0.5:
            dim = max(8, dim // 8 * 8)
        rows = _log(rng, 1, max(2, min(524288, (1 << 27) // dim)))
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype,
                "wdtype": rng.choice(["float32", dtype, "none"]), "train": rng.random() < 0.7}
    if op == "scan":
        steps = _log(rng, 1, 65536)
        dim = _log(rng, 1, min(2048, (1 << 25) // steps))
        if rng.random() < 0.5:
            dim = max(8, dim // 8 * 8)
        batch = _log(rng, 1, max(2, min(65536, (1 << 26) // (steps * dim))))
        return {"op": op, "steps": steps, "batch": batch, "dim": dim, "dtype": dtype, "gated": rng.random() < 0.6,
                "resets": rng.random() < 0.5, "padded": rng.random() < 0.4, "initial": rng.random() < 0.5,
                "batch_first": rng.random() < 0.4, "train": rng.random() < 0.7}
    if op == "step":
        dim = _log(rng, 1, 2048)
        return {"op": op, "batch": _log(rng, 1, max(2, min(131072, (1 << 24) // dim))), "dim": dim, "dtype": dtype,
                "gated": rng.random() < 0.6, "resets": rng.random() < 0.5}
    hidden = _log(rng, 8, 4096)
    layers = rng.randint(1, max(1, min(120, (1 << 26) // (hidden * hidden))))
    return {"op": op, "towers": rng.choice([1, 2]), "dim": _log(rng, 8, 512), "hidden": hidden, "layers": layers,
            "out": _log(rng, 1, 128), "dtype": dtype, "bits": rng.choice([8, 32]),
            "master": dtype != "float32" and rng.random() < 0.6, "clip": rng.choice([0.0, 0.5, 100.0])}


# ---------------------------------------------------------------------------- inputs

def _shapes(case):
    shapes = []
    for _ in range(case["towers"]):
        last = case["dim"]
        for _ in range(case["layers"]):
            shapes += [(case["hidden"], last), (case["hidden"],)]
            last = case["hidden"]
        shapes += [(case["out"], last), (case["out"],)]
    return shapes


def _places(shapes):
    """(first element, element count) of each tensor in the flat buffers, and their length."""
    places, at = [], 0
    for shape in shapes:
        n = math.prod(shape)
        places.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return places, at


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    if op == "norm":
        rows, dim = case["rows"], case["dim"]
        # hidden activations: every row with a mean and a spread of its own
        x = _normal(gen, rows, dim) * (0.3 + 2 * torch.rand(rows, 1, device="cuda", generator=gen))
        x += _normal(gen, rows, 1)
        state = {"case": case, "x": x.to(dtype), "w": None, "b": None}
        if case["wdtype"] != "none":
            wdtype = DTYPES[case["wdtype"]]
            state["w"] = (1 + 0.2 * _normal(gen, dim)).to(wdtype)
            state["b"] = (0.2 * _normal(gen, dim)).to(wdtype)
        if case["train"]:
            state["dy"] = _normal(gen, rows, dim).to(dtype)
            for k in ("x", "w", "b"):
                if state[k] is not None:
                    state[k].requires_grad_()
        return state
    if op == "scan":
        steps, batch, dim = case["steps"], case["batch"], case["dim"]

        def tensor(values):
            return values.to(dtype).transpose(0, 1) if case["batch_first"] else values.to(dtype)

        shape = (batch, steps, dim) if case["batch_first"] else (steps, batch, dim)
        gate = _normal(gen, *shape) + 2                    # a memory of about eight steps
        if not case["gated"]:
            gate = torch.sigmoid(gate) * torch.where(torch.rand(*shape, device="cuda", generator=gen) < 0.1, -1.0, 1.0)
        state = {"case": case, "gate": tensor(gate), "x": tensor(_normal(gen, *shape)), "h0": None, "reset": None,
                 "lengths": None}
        del gate
        if case["initial"]:
            state["h0"] = _normal(gen, batch, dim)
        if case["resets"]:
            state["reset"] = torch.rand(steps, batch, device="cuda", generator=gen) < RESET_RATE
        if case["padded"]:
            n = torch.rand(batch, device="cuda", generator=gen) * 1.1 - 0.1    # about one in eleven is empty
            state["lengths"] = (n.clamp_(0, 1) * steps).round().long()
        if case["train"]:
            state["dh"] = tensor(_normal(gen, *shape))
            state["dhn"] = _normal(gen, batch, dim)
            for k in ("gate", "x", "h0"):
                if state[k] is not None:
                    state[k].requires_grad_()
        return state
    if op == "step":
        batch, dim = case["batch"], case["dim"]
        gate = _normal(gen, batch, dim) + 2
        if not case["gated"]:
            gate = torch.sigmoid(gate)
        return {"case": case, "gate": gate.to(dtype), "x": _normal(gen, batch, dim).to(dtype),
                "h": _normal(gen, batch, dim),
                "reset": torch.rand(batch, device="cuda", generator=gen) < RESET_RATE if case["resets"] else None}
    # adamw: parameters, gradients and moments, each in one flat buffer
    shapes = _shapes(case)
    places, total = _places(shapes)
    p = torch.zeros(total, device="cuda")
    g = torch.zeros(total, device="cuda")
    m = torch.zeros(total, device="cuda")
    v = torch.zeros(total, device="cuda")
    for (at, n), shape in zip(places, shapes):
        size = 10 ** (3 * float(torch.rand((), generator=torch.Generator().manual_seed(seed + at))) - 4)
        p[at:at + n] = _normal(gen, n) / math.sqrt(shape[-1])
        g[at:at + n] = _normal(gen, n) * size
        m[at:at + n] = _normal(gen, n) * (0.3 * size)
        v[at:at + n] = (size * (0.5 + torch.rand(n, device="cuda", generator=gen))) ** 2
    state = {"case": case, "p": p.to(dtype), "g": g.to(dtype), "done": torch.full((), STEPS_DONE, device="cuda",
                                                                                  dtype=torch.float64)}
    moments = {}
    if case["master"]:
        # masters lie between their parameters and the parameters' neighbours
        moments["master"] = state["p"].float() * (1 + (torch.finfo(dtype).eps / 8) *
                                                  torch.rand(total, device="cuda", generator=gen))
    if case["bits"] == 8:
        for name, values, code in (("exp_avg", m, torch.float8_e4m3fn), ("exp_avg_sq", v, torch.float8_e5m2)):
            scale = values.view(-1, BLOCK).abs().amax(1) / torch.finfo(code).max
            scale.clamp_(min=torch.finfo(torch.float32).tiny)
            moments[name] = (values.view(-1, BLOCK) / scale.unsqueeze(1)).view(-1).to(code)
            moments[name + "_scale"] = scale
    else:
        moments["exp_avg"], moments["exp_avg_sq"] = m, v
    state["moments"] = moments
    state["opt"] = _optimizer(case, state, shapes, places) if own else None
    return state


def _optimizer(case, state, shapes, places):
    """The framework's optimiser over views of the flat parameters, its moments set to the state's."""
    params = []
    for (at, n), shape in zip(places, shapes):
        t = state["p"][at:at + n].view(shape).requires_grad_()
        t.grad = state["g"][at:at + n].view(shape)
        params.append(t)
    opt = _package("optim").AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY,
                                  state_bits=case["bits"], max_grad_norm=case["clip"] or None,
                                  master_weights=case["master"], seed=SEED)
    buffers = opt.state_buffers()[0]
    for name, values in state["moments"].items():
        buffers[name].copy_(values)
    buffers["step"].fill_(STEPS_DONE)
    state["moments"] = {name: buffers[name] for name in state["moments"]}
    return opt


# ---------------------------------------------------------------------------- one pass

def run(state):
    return {"norm": _run_norm, "scan": _run_scan, "step": _run_step, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_norm(s):
    train = s["case"]["train"]
    if own:
        y = _package("layernorm").layer_norm(s["x"], s["w"], s["b"], EPS)
        if not train:
            return {"y": y}
        leaves = [k for k in ("x", "w", "b") if s[k] is not None]
        grads = torch.autograd.grad(y, [s[k] for k in leaves], s["dy"])
        return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}
    with torch.no_grad():
        x = s["x"].float()
        centred = x - x.mean(1, keepdim=True)
        rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
        xhat = centred * rstd
        y = xhat if s["w"] is None else xhat * s["w"].float() + s["b"].float()
        out = {"y": y.to(s["x"].dtype)}
        if train:
            dy = s["dy"].float()
            g = dy if s["w"] is None else dy * s["w"].float()
            dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
            out["dx"] = dx.to(s["x"].dtype)
            if s["w"] is not None:
                out["dw"] = (dy * xhat).sum(0).to(s["w"].dtype)
                out["db"] = dy.sum(0).to(s["b"].dtype)
        return out


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = 0 along the first axis, by doubling."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _run_scan(s):
    case = s["case"]
    if own:
        rec = _package("recurrence")
        h, hn = (rec.gated_scan if case["gated"] else rec.linear_scan)(s["gate"], s["x"], s["h0"], reset=s["reset"],
                                                                       lengths=s["lengths"])
        if not case["train"]:
            return {"h": h, "hn": hn}
        leaves = [k for k in ("gate", "x", "h0") if s[k] is not None]
        grads = torch.autograd.grad([h, hn], [s[k] for k in leaves], [s["dh"], s["dhn"]])
        return {"h": h.detach(), "hn": hn.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}
    with torch.no_grad():
        gate, x = s["gate"].float(), s["x"].float()
        f = torch.sigmoid(gate) if case["gated"] else gate
        keep = torch.sigmoid(-gate) if case["gated"] else None          # 1 - f
        a, b = f, (keep * x if case["gated"] else x)
        live = None
        if s["reset"] is not None:
            a = torch.where(s["reset"].unsqueeze(2), 0.0, a)
        if s["lengths"] is not None:
            t = torch.arange(case["steps"], device=x.device)
            live = (t.unsqueeze(1) < s["lengths"].unsqueeze(0)).unsqueeze(2)
            a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
        if s["h0"] is not None:
            b = torch.cat([b[:1] + a[:1] * s["h0"], b[1:]])
        h = _prefix(a, b)
        out = {"h": (h if live is None else torch.where(live, h, 0.0)).to(s["x"].dtype), "hn": h[-1].clone()}
        if not case["train"]:
            return out
        dh = s["dh"].float() if live is None else torch.where(live, s["dh"].float(), 0.0)
        dh = torch.cat([dh[:-1], dh[-1:] + s["dhn"]])
        g = _prefix(torch.cat([a[1:], a.new_zeros(1, *a.shape[1:])]).flip(0), dh.flip(0)).flip(0)
        first = h.new_zeros(1, *h.shape[1:]) if s["h0"] is None else s["h0"].unsqueeze(0)
        before = torch.cat([first, h[:-1]])
        if s["reset"] is not None:
            before = torch.where(s["reset"].unsqueeze(2), 0.0, before)
        dx = g * keep if case["gated"] else g
        dgate = g * (before - x) * f * keep if case["gated"] else g * before
        if live is not None:
            dx, dgate = torch.where(live, dx, 0.0), torch.where(live, dgate, 0.0)
        out["dgate"], out["dx"] = dgate.to(s["gate"].dtype), dx.to(s["x"].dtype)
        if s["h0"] is not None:
            out["dh0"] = g[0] * a[0]
        return out


def _run_step(s):
    case = s["case"]
    if own:
        rec = _package("recurrence")
        h = (rec.gated_step if case["gated"] else rec.linear_step)(s["gate"], s["x"], s["h"], reset=s["reset"])
        return {"h": h, "state": s["h"]}
    gate, x = s["gate"].float(), s["x"].float()
    before = s["h"] if s["reset"] is None else torch.where(s["reset"].unsqueeze(1), 0.0, s["h"])
    if case["gated"]:
        new = torch.sigmoid(gate) * before + torch.sigmoid(-gate) * x
    else:
        new = gate * before + x
    s["h"].copy_(new)
    return {"h": new.to(s["x"].dtype), "state": s["h"]}


def _shifted(z, n):
    """Logical right shift of the 64 bits of z."""
    return (z >> n) & ((1 << (64 - n)) - 1)


def _mix(z):
    """The finaliser of the splitmix64 generator on int64 tensors (products wrap)."""
    z = z + (0x9E3779B97F4A7C15 - (1 << 64))
    z = (z ^ _shifted(z, 30)) * (0xBF58476D1CE4E5B9 - (1 << 64))
    z = (z ^ _shifted(z, 27)) * (0x94D049BB133111EB - (1 << 64))
    return z ^ _shifted(z, 31)


def _draws(step, total, device):
    """The 16-bit uniform numbers in [0, 1) that round both moments of every element in step `step`."""
    key = _mix(torch.full((), SEED, dtype=torch.int64, device=device) ^ _mix(step.long()))
    words = _mix(key + torch.arange(total // 2, device=device))
    parts = torch.stack([_shifted(words, k) & 0xFFFF for k in (0, 16, 32, 48)], 1).to(torch.float64) / 65536
    return parts[:, 0::2].reshape(-1), parts[:, 1::2].reshape(-1)


def _coded(values, u, dtype, least):
    """Values as codes of an 8-bit type and a scale for each BLOCK, rounded away from zero where u and what
    is left over of a step make a whole one; `least`: positive values stay above zero."""
    finfo = torch.finfo(dtype)
    rows = values.view(-1, BLOCK)
    scale = (rows.abs().amax(1) / finfo.max).clamp(min=torch.finfo(torch.float32).tiny)
    size = (rows.double().abs() / scale.unsqueeze(1).double()).clamp(max=finfo.max).view(-1)
    steps = torch.ldexp(torch.full_like(size, finfo.eps), torch.frexp(size.clamp(min=finfo.tiny)).exponent - 1)
    code = torch.floor(size / steps + u) * steps
    if least:
        code = torch.where(size > 0, code.clamp(min=finfo.tiny * finfo.eps), code)
    return torch.copysign(code, values.double()).to(dtype), scale


def _run_adamw(s):
    case, q = s["case"], s["moments"]
    if own:
        s["opt"].step()
        return {"p": s["p"], **q}
    s["done"] += 1
    g = s["g"].float()
    if case["clip"]:
        norm = torch.sqrt(torch.sum(g.square(), dtype=torch.float64))
        g = g * (case["clip"] / (norm + 1e-6)).clamp(max=1.0).float()
    m, v = q["exp_avg"].float(), q["exp_avg_sq"].float()
    if case["bits"] == 8:
        m = (m.view(-1, BLOCK) * q["exp_avg_scale"].unsqueeze(1)).view(-1)
        v = (v.view(-1, BLOCK) * q["exp_avg_sq_scale"].unsqueeze(1)).view(-1)
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g.square()
    first, second = 1 - BETA1 ** s["done"], 1 - BETA2 ** s["done"]
    p = q["master"] if case["master"] else s["p"].float()
    p = p * (1 - LR * DECAY) - (LR / first).float() * m / (torch.sqrt(v) / torch.sqrt(second).float() + ADAM_EPS)
    s["p"].copy_(p)
    if case["master"]:
        q["master"].copy_(p)
    if case["bits"] == 8:
        um, uv = _draws(s["done"], p.numel(), p.device)
        for name, values, u in (("exp_avg", m, um), ("exp_avg_sq", v, uv)):
            code, scale = _coded(values, u, q[name].dtype, name == "exp_avg_sq")
            q[name].copy_(code)
            q[name + "_scale"].copy_(scale)
    else:
        q["exp_avg"].copy_(m)
        q["exp_avg_sq"].copy_(v)
    return {"p": s["p"], **q}


# ---------------------------------------------------------------------------- the work of a pass

def work(case):
    size = DTYPES[case["dtype"]].itemsize
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["dim"]
        w = 0 if case["wdtype"] == "none" else 2 * case["dim"] * DTYPES[case["wdtype"]].itemsize
        if case["train"]:       # x, dy in; y, dx out; weight and bias in, their gradients out
            return {"bytes": 4 * n * size + 2 * w, "flops": 20 * n}
        return {"bytes": 2 * n * size + w, "flops": 8 * n}
    if op in ("scan", "step"):
        rows = case.get("steps", 1) * case["batch"]
        n, c = rows * case["dim"], case["batch"] * case["dim"]
        extra = rows if case["resets"] else 0
        if op == "step":        # gate, x in, h out, the state in and out
            return {"bytes": 3 * n * size + 8 * c + extra, "flops": (8 if case["gated"] else 2) * n}
        extra += 4 * c * (1 + case["initial"]) + 8 * case["batch"] * case["padded"]
        if case["train"]:       # gate, x, dh in; h, dgate, dx out
            return {"bytes": 6 * n * size + 2 * extra, "flops": (24 if case["gated"] else 6) * n}
        return {"bytes": 3 * n * size + extra, "flops": (8 if case["gated"] else 2) * n}
    n = sum(math.prod(shape) for shape in _shapes(case))
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * size + moments + (8 if case["master"] else 0)), "flops": 16 * n}


# ---------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "scan": _exact_scan, "step": _exact_step, "adamw": _exact_adamw}[case["op"]](s)


def _exact_norm(s):
    x = s["x"].double()
    dim = x.shape[1]
    mean = x.sum(1) / dim
    spread = torch.sqrt(((x - mean[:, None]) ** 2).sum(1) / dim + EPS)
    z = (x - mean[:, None]) / spread[:, None]
    w = torch.ones(dim, dtype=torch.float64, device=x.device) if s["w"] is None else s["w"].double()
    out = {"y": z * w if s["b"] is None else z * w + s["b"].double()}
    if s["case"]["train"]:
        dy = s["dy"].double()
        # dx = (I - 1/n 11^T - 1/n z z^T) (w dy) / spread
        u = dy * w
        out["dx"] = (u - (u.sum(1) / dim)[:, None] - z * (torch.einsum("rd,rd->r", u, z) / dim)[:, None]) / spread[:, None]
        if s["w"] is not None:
            out["dw"], out["db"] = torch.einsum("rd,rd->d", dy, z), torch.einsum("rd->d", dy)
    return out


def _exact_scan(s):
    """Step by step, forward in time and back."""
    case = s["case"]
    steps, batch, dim = case["steps"], case["batch"], case["dim"]
    zero = torch.zeros(batch, dim, dtype=torch.float64, device="cuda")
    ones = torch.ones(steps, batch, 1, dtype=torch.float64, device="cuda")
    live = ones if s["lengths"] is None else (torch.arange(steps, device="cuda")[:, None, None] <
                                              s["lengths"][None, :, None]).double()
    pass_on = ones if s["reset"] is None else 1 - s["reset"].double()[:, :, None]
    f = s["gate"].double()
    if case["gated"]:
        f = 1 / (1 + torch.exp(-f))
        into = 1 / (1 + torch.exp(s["gate"].double()))
    else:
        into = None
    x = s["x"].double()
    # h_t = carry_t h_{t-1} + inflow_t
    carry = f * pass_on * live + (1 - live)
    inflow = (x if into is None else into * x) * live
    start = zero if s["h0"] is None else s["h0"].double()
    states = torch.empty(steps + 1, batch, dim, dtype=torch.float64, device="cuda")
    states[0] = start
    for t in range(steps):
        torch.addcmul(inflow[t], carry[t], states[t], out=states[t + 1])
    out = {"h": states[1:] * live, "hn": states[steps].clone()}
    if not case["train"]:
        return out
    flow = s["dh"].double() * live
    down = torch.empty(steps + 1, batch, dim, dtype=torch.float64, device="cuda")
    down[steps] = s["dhn"].double()
    into_state = torch.empty(steps, batch, dim, dtype=torch.float64, device="cuda")
    for t in range(steps - 1, -1, -1):
        torch.add(flow[t], down[t + 1], out=into_state[t])
        torch.mul(carry[t], into_state[t], out=down[t])
    before = states[:-1] * pass_on
    if case["gated"]:
        out["dgate"] = into_state * (before - x) * f * into * live
        out["dx"] = into_state * into * live
    else:
        out["dgate"], out["dx"] = into_state * before * live, into_state * live
    if s["h0"] is not None:
        out["dh0"] = down[0].clone()
    return out


def _exact_step(s):
    before = s["h"].double()
    if s["reset"] is not None:
        before = before * (1 - s["reset"].double()[:, None])
    a, x = s["gate"].double(), s["x"].double()
    if s["case"]["gated"]:
        f = 1 / (1 + torch.exp(-a))
        new = f * before + x / (1 + torch.exp(a))
    else:
        new = a * before + x
    return {"h": new, "state": new.clone()}


def _exact_rounding(step, count):
    """(count / 2, 4) numbers below 2^16: of each pair of elements the first's for both moments, then the second's."""
    def mixed(z):
        z = z - 7046029254386353131
        for right, factor in ((30, -4658895280553007687), (27, -7723592293110705685)):
            z = (z ^ ((z >> right) & (2 ** (64 - right) - 1))) * factor
        return z ^ ((z >> 31) & (2 ** 33 - 1))

    key = mixed(SEED ^ mixed(torch.tensor(step, device="cuda")))
    return mixed(torch.arange(count // 2, device="cuda") + key).view(torch.int16).view(-1, 4).long() & 65535


def _exact_codes(values, number, code, least):
    """The 8-bit type's neighbours of each value in units of its block's scale, one of them chosen."""
    top = torch.finfo(code).max
    scale = (values.abs().view(-1, BLOCK).max(1).values / top).clamp(min=torch.finfo(torch.float32).tiny)
    units = (values / scale.repeat_interleave(BLOCK)).abs().clamp(max=top)
    near = units.to(code)
    low = torch.where(near.double() > units, near.view(torch.uint8) - 1, near.view(torch.uint8))
    below = low.view(code).double()
    above = (low + 1).view(code).double()
    up = (units > below) & ((units - below) / (above - below) + number / 65536.0 >= 1)
    chosen = torch.where(up, above, below)
    if least:
        chosen = torch.where((units > 0) & (chosen == 0), above, chosen)
    return torch.where(values < 0, -chosen, chosen), scale


def _exact_adamw(s):
    case, q = s["case"], s["moments"]
    t = STEPS_DONE + 1
    grad = s["g"].double()
    if case["clip"]:
        grad = grad * min(1.0, case["clip"] / (math.sqrt(float((grad ** 2).sum())) + 1e-6))

    def moment(name):
        values = q[name].double()
        if case["bits"] == 8:
            values = values * q[name + "_scale"].double().repeat_interleave(BLOCK)
        return values

    first = moment("exp_avg") * BETA1 + grad * (1 - BETA1)
    second = moment("exp_avg_sq") * BETA2 + grad ** 2 * (1 - BETA2)
    p = (q["master"] if case["master"] else s["p"]).double()
    rate = first / (1 - BETA1 ** t) / (torch.sqrt(second / (1 - BETA2 ** t)) + ADAM_EPS)
    p = p - LR * DECAY * p - LR * rate
    out = {"p": p, "exp_avg": first, "exp_avg_sq": second}
    if case["master"]:
        out["master"] = p.clone()
    if case["bits"] == 8:
        draws = _exact_rounding(t, p.numel())
        for k, name in enumerate(("exp_avg", "exp_avg_sq")):
            out[name], out[name + "_scale"] = _exact_codes(out[name], draws[:, k::2].reshape(-1), q[name].dtype, k == 1)
    return out
