"""The layer norm entries with the mean in two parts refuse what the others do, without a GPU."""
import ctypes as C

from conftest import pkg_module


def test_refusals():
    lib = pkg_module("_lib").load()
    keep = (C.c_double * 512)()
    p = C.cast(keep, C.c_void_p)
    fwd = lambda m=p, rest=p, r=p, rows=2, y=p: lib.f16_layer_norm_fwd_rest(p, rows, 8, 8, 2, None, None, 2, 1e-5, y, 8, m,
                                                                            rest, r, None)
    assert fwd(m=None) == 1 and fwd(r=None) == 1 and fwd(rows=0) == 1 and fwd(y=None) == 1
    assert fwd(m=None, r=None) == 1                            # a rest of no mean
    bwd = lambda m=p, r=p, s=p, n=16: lib.f16_layer_norm_bwd_rest(p, 8, p, 8, 2, 8, 2, None, 2, m, p, r, p, 8, p, None, s, n, None)
    assert bwd(m=None) == 1 and bwd(r=None) == 1 and bwd(s=None) == 1 and bwd(n=15) == 1
