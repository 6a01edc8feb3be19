"""Host side of the training operators, without a GPU: the C entry points refuse bad arguments before any
launch, the ctypes mirrors have the header's layout, and the Python wrappers refuse CPU tensors (there is
no fallback) where torch's modules take over where they are documented to."""
import ctypes as C
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT, pkg_module

ARG, ALIGN, TOO_LARGE = 1, 2, 6


@pytest.fixture()
def buf():
    b = (C.c_double * 512)()
    return C.cast(b, C.c_void_p), b


def test_layer_norm_entries_refuse(buf):
    lib = pkg_module("_lib").load()
    p, _keep = buf
    fwd = lambda x=p, rows=2, cols=8, ldx=8, dt=2, w=None, b=None, wdt=2, eps=1e-5, y=p, ldy=8, m=None, r=None: \
        lib.f16_layer_norm_fwd(x, rows, cols, ldx, dt, w, b, wdt, eps, y, ldy, m, r, None)
    assert fwd(x=None) == ARG and fwd(y=None) == ARG and fwd(rows=0) == ARG and fwd(cols=0) == ARG
    assert fwd(ldx=-1) == ARG and fwd(ldy=7) == ARG and fwd(dt=3) == ARG and fwd(wdt=-1) == ARG
    assert fwd(m=p) == ARG                                     # one of the two statistics
    assert fwd(eps=-1.0) == ARG and fwd(eps=float("nan")) == ARG
    assert fwd(x=C.c_void_p(p.value + 2)) == ALIGN and fwd(dt=0, x=C.c_void_p(p.value + 1)) == ALIGN
    bwd = lambda dy=p, x=p, rows=2, cols=8, dt=2, m=p, r=p, dx=p, dw=p, s=p, n=16: \
        lib.f16_layer_norm_bwd(dy, 8, x, 8, rows, cols, dt, None, 2, m, r, dx, 8, dw, None, s, n, None)
    assert bwd(dy=None) == ARG and bwd(m=None) == ARG and bwd(rows=0) == ARG and bwd(dt=9) == ARG
    assert bwd(s=None) == ARG and bwd(n=15) == ARG             # no room for one block's sums
    assert bwd(dx=None, dw=None) == 0                          # nothing wanted
    assert fwd(cols=2 ** 29 + 1, ldy=2 ** 30) == TOO_LARGE
    assert lib.f16_layer_norm_scratch_floats(0, 8) == 0
    assert lib.f16_layer_norm_scratch_floats(3, 8) == 2 * 8 * 3


def test_scan_entries_refuse(buf):
    _lib = pkg_module("_lib")
    lib = _lib.load()
    p, _keep = buf
    ok = dict(dtype=2, gated=1, steps=3, batch=2, dim=4, gate=p.value, x=p.value, h=p.value, saved=p.value, dh=p.value)

    def call(fn, **change):
        a = _lib.ScanArgs()
        for k, v in {**ok, **change}.items():
            setattr(a, k, v)
        return fn(C.byref(a), None)

    for fn in (lib.f16_scan_fwd, lib.f16_scan_bwd):
        assert fn(None, None) == ARG
        for change in (dict(gate=None), dict(x=None), dict(steps=0), dict(batch=-1), dict(dim=0), dict(dtype=3),
                       dict(reset=p.value, reset_bytes=2)):
            assert call(fn, **change) == ARG
        assert call(fn, steps=2 ** 31) == TOO_LARGE
        assert call(fn, x=p.value + 2) == ALIGN
        assert call(fn, reset=p.value + 1, reset_bytes=4) == ALIGN
        assert call(fn, scratch=p.value + 4) == ALIGN
        assert call(fn, batch=2 ** 40, dim=2 ** 40) == TOO_LARGE
    assert call(lib.f16_scan_fwd, h=None) == ARG
    assert call(lib.f16_scan_bwd, saved=None) == ARG and call(lib.f16_scan_bwd, dh=None) == ARG
    assert lib.f16_scan_saved_floats(17, 2, 3) == 2 * 6 and lib.f16_scan_saved_floats(0, 2, 3) == 0
    # one chunk, or channels enough for every SM: time is not cut; else three floats a segment and channel
    assert lib.f16_scan_scratch_floats(16, 1, 8) == 0 and lib.f16_scan_scratch_floats(64, 16384, 128) == 0
    assert lib.f16_scan_scratch_floats(32, 1, 8) == 3 * 2 * 8 and lib.f16_scan_scratch_floats(-1, 1, 8) == 0
    step = lambda gate=p, state=p, dt=2, sb=4, hb=4, batch=2, rb=0, reset=None: \
        lib.f16_scan_step(gate, 4, p, 4, batch, 4, dt, 1, reset, rb, 1, state, sb, p, hb, None)
    assert step(gate=None) == ARG and step(state=None) == ARG and step(batch=0) == ARG and step(dt=5) == ARG
    assert step(sb=3) == ARG and step(hb=3) == ARG and step(reset=p, rb=8) == ARG
    assert step(state=C.c_void_p(p.value + 2)) == ALIGN


def test_adamw_entries_refuse(buf):
    _lib = pkg_module("_lib")
    lib = _lib.load()
    p, _keep = buf
    used = C.c_int(0)
    one = (C.c_void_p * 1)(p.value)
    n1, n0 = (C.c_int64 * 1)(4), (C.c_int64 * 1)(0)
    odd = (C.c_void_p * 1)(p.value + 2)
    assert lib.f16_grad_squares(0, one, n1, 2, p, 1, C.byref(used), None) == ARG
    assert lib.f16_grad_squares(1, one, n0, 2, p, 1, C.byref(used), None) == ARG
    assert lib.f16_grad_squares(1, one, n1, 7, p, 1, C.byref(used), None) == ARG
    assert lib.f16_grad_squares(1, odd, n1, 2, p, 1, C.byref(used), None) == ALIGN
    assert lib.f16_grad_squares(1, one, n1, 2, p, 0, C.byref(used), None) == TOO_LARGE
    first, off = (C.c_int64 * 1)(256), (C.c_int64 * 1)(100)
    index = (C.c_int32 * 1)(0)
    at = C.addressof
    ok = dict(count=1, dtype=2, state_bits=32, params_host=at(one), grads_host=at(one), numel_host=at(n1),
              first_host=at(first), index_host=at(index), exp_avg=p.value, exp_avg_sq=p.value, steps=p.value, ticket=p.value)

    def call(**change):
        a = _lib.AdamwArgs()
        for k, v in {**ok, **change}.items():
            setattr(a, k, v)
        return lib.f16_adamw_step(C.byref(a), None)

    assert lib.f16_adamw_step(None, None) == ARG
    for change in (dict(count=0), dict(dtype=4), dict(state_bits=16), dict(state_bits=8), dict(params_host=None),
                   dict(steps=None), dict(ticket=None), dict(numel_host=at(n0)), dict(first_host=at(off)),
                   dict(master=p.value), dict(partial=p.value, partials=0)):
        assert call(**change) == ARG, change
    assert call(grads_host=at(odd)) == ALIGN and call(exp_avg=p.value + 4) == ALIGN


PAIRS = [("f16_scan_args", "ScanArgs"), ("f16_adamw_args", "AdamwArgs")]


def test_struct_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    _lib = pkg_module("_lib")
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "f16env.h"', "int main(void) {"]
    for cname, cls in PAIRS:
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in getattr(_lib, cls)._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([cc, "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    said = {}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, key, value = line.split()
        said[name, key] = int(value)
    for cname, cls in PAIRS:
        py = getattr(_lib, cls)
        assert C.sizeof(py) == said[cname, "size"]
        assert all(getattr(py, f[0]).offset == said[cname, f[0]] for f in py._fields_)


def test_constants_match_the_header():
    text = (ROOT / "include" / "f16env.h").read_text()
    define = lambda n: int(text.split(f"#define {n} ")[1].split()[0])
    _lib = pkg_module("_lib")
    assert _lib.DTYPES == {torch.bfloat16: define("F16_DTYPE_BF16"), torch.float16: define("F16_DTYPE_FP16"),
                           torch.float32: define("F16_DTYPE_FP32")}
    assert pkg_module("optim").BLOCK == define("F16_ADAMW_BLOCK")
    assert pkg_module("recurrence").CHUNK == define("F16_SCAN_CHUNK")
    assert pkg_module("layernorm").MAX_DIM == 2 ** 29


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 2, 8)
    with pytest.raises(ValueError):
        pkg_module("layernorm").layer_norm(x)
    with pytest.raises(ValueError):
        pkg_module("recurrence").gated_scan(x, x)
    with pytest.raises(ValueError):
        pkg_module("recurrence").gated_step(x[0], x[0], x[0])
    with pytest.raises(ValueError):
        pkg_module("optim").AdamW([torch.zeros(3, requires_grad=True)])


def test_layer_norm_module_on_cpu_is_torchs():
    ln, sm = pkg_module("layernorm"), pkg_module("splitmm")
    torch.manual_seed(0)
    mine, ref = ln.LayerNorm(24, eps=1e-3), torch.nn.LayerNorm(24, eps=1e-3)
    torch.nn.init.normal_(mine.weight)
    ref.load_state_dict(mine.state_dict())
    x = torch.randn(5, 24)
    assert torch.equal(mine(x), ref(x))
    with pytest.raises(ValueError):
        ln.LayerNorm((4, 6))
    net = torch.nn.Sequential(torch.nn.Linear(24, 64), ln.LayerNorm(64), torch.nn.Tanh(), torch.nn.Linear(64, 3))
    assert torch.equal(sm.run_tower(net, x), net(x))


def test_trainer_names_its_optimiser():
    tr = pkg_module("trainer")
    params = [torch.zeros(3, requires_grad=True)]
    assert isinstance(tr.make_optimizer(params, 1e-3, tr.PPOConfig()), torch.optim.Adam)
    with pytest.raises(ValueError):
        tr.make_optimizer(params, 1e-3, tr.PPOConfig(optimizer="sgd"))
    with pytest.raises(ValueError):
        tr.make_optimizer(params, 1e-3, tr.PPOConfig(optimizer="adamw"))        # CPU parameters
