"""Refusals of the serving ops' C entries that need no device: pointers off their elements' boundary, at which a
kernel's loads would fault."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def S():
    from xdna_engine_b200 import _build, serving
    _build.build()
    return serving


def test_pointers_off_their_elements(S):
    import xdna_engine_b200 as X
    L = S._lib()
    room = (C.c_double * 64)()
    p = (C.addressof(room) + 15) // 16 * 16
    norm = dict(x=p, x_f32=1, xs=16, res=p, rf=0, rs=16, g=p, u=0, eps=1e-6, M=0, D=16, ro=p, y=p, q=p, s=p, st=None)
    assert L.xdna_rmsnorm_residual_i8(*norm.values()) == 0
    for bad in (dict(x=p + 2), dict(x=p + 1, x_f32=0), dict(res=p + 1), dict(res=p + 2, rf=1), dict(ro=p + 1),
                dict(g=p + 2), dict(y=p + 1), dict(s=p + 2)):
        assert L.xdna_rmsnorm_residual_i8(*{**norm, **bad}.values()) == -1 and "aligned" in X.last_error(), bad
    logits = dict(x=p, f=1, ls=8, B=0, V=8, h=p, nh=4, hs=p, np=p, rep=p, fr=p, pr=p, bi=p, b=p, nb=4, bs=p, m=p, ms=1,
                  o=p + 32, os=8, ids=p, ws=p, st=None)
    assert L.xdna_logits_process(*logits.values()) == 0
    for name in ("x", "h", "hs", "np", "rep", "fr", "pr", "bi", "b", "bs", "m", "o"):
        assert L.xdna_logits_process(*{**logits, name: p + 2}.values()) == -1 and "aligned" in X.last_error(), name
    assert L.xdna_logits_process(*{**logits, "ids": p + 4}.values()) == -1 and "aligned" in X.last_error()
    assert L.xdna_logits_process(*{**logits, "x": p + 1, "f": 0}.values()) == -1 and "aligned" in X.last_error()
    assert L.xdna_logits_process(*{**logits, "x": p + 2, "f": 0}.values()) == 0
