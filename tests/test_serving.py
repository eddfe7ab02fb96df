"""The serving ops' refusals that need no device: NULL arguments and impossible shapes at the C
ABI, and tensors that are not on the cache's GPU."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def S():
    from xdna_engine_b200 import _build, serving
    _build.build()
    return serving


def test_null_and_shape_refusals(S):
    import xdna_engine_b200 as X
    L = S._lib()
    one = (C.c_float * 64)()
    p = C.addressof(one)
    assert L.xdna_paged_cache_create(None, None) is None
    assert "null" in X.last_error()
    assert L.xdna_paged_append(None, 0, 1, 1, 0, p, 64, p, 64, p, 64, None, p, p, 1, 1, 1, None, 0, 0, 0, p, None) == -1
    assert "null" in X.last_error()
    assert L.xdna_paged_attention(None, 0, p, 64, 1, p, 1, 1, 1, p, 0.125, 0, p, None, None) == -1
    assert L.xdna_paged_cache_check(None, None) == -1
    L.xdna_paged_cache_free(None)
    norm = lambda **k: L.xdna_rmsnorm_residual_i8(*{**dict(  # noqa: E731
        x=p, x_f32=1, xs=16, res=None, rf=1, rs=16, g=p, u=0, eps=1e-6, M=1, D=16, ro=None, y=None, q=p, s=p,
        st=None), **k}.values())
    for bad, why in ((dict(x=None), "null"), (dict(g=None), "null"), (dict(q=None), "together"),
                     (dict(s=None), "together"), (dict(q=None, s=None), "no output"), (dict(D=0), "D outside"),
                     (dict(D=16385), "D outside"), (dict(M=-1), "negative M"), (dict(xs=15), "stride"),
                     (dict(res=p, rs=15), "stride"), (dict(eps=-1e-6), "eps")):
        assert norm(**bad) == -1 and why in X.last_error(), bad
    assert norm(M=0) == 0
    logits = lambda **k: L.xdna_logits_process(*{**dict(  # noqa: E731
        x=p, f=1, ls=8, B=2, V=8, h=None, nh=0, hs=None, np=None, rep=None, fr=None, pr=None, bi=None, b=None, nb=0,
        bs=None, m=None, ms=0, o=p, os=8, ids=p, ws=p, st=None), **k}.values())
    for bad, why in ((dict(x=None), "null"), (dict(o=None), "null"), (dict(V=0), "V"), (dict(B=-1), "B"),
                     (dict(h=p), "together"), (dict(hs=p), "together"), (dict(rep=p), "history"),
                     (dict(np=p), "history"), (dict(b=p), "together"), (dict(bi=p, b=p), "together"),
                     (dict(ls=7), "stride"), (dict(os=7), "stride"), (dict(m=p, ms=0), "mask_stride"),
                     (dict(nh=-1), "n_history"), (dict(nb=-1), "n_biases"), (dict(f=0), "bf16"),
                     (dict(os=16), "stride"), (dict(ws=None, B=1, V=200000, ls=200000, os=200000), "workspace"), (dict(B=65536), "65535")):
        assert logits(**bad) == -1 and why in X.last_error(), bad
    assert logits(B=0) == 0


def test_tensors_elsewhere(S):
    class Dev:
        ordinal, handle = 0, None

    pool = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="not on device 0"):
        S.PagedCache(Dev, pool, pool.clone())
    with pytest.raises(ValueError):
        S.PagedCache(Dev, pool[0], pool[0])


def test_rope_table(S):
    import math
    t = S.rope_table(5, 8, theta=100.0, device="cpu")
    assert t.shape == (5, 8) and t.dtype == torch.float32
    for p in range(5):
        for i in range(4):
            a = p * 100.0 ** (-2 * i / 8)
            assert t[p, i] == torch.tensor(math.cos(a)).float() and abs(float(t[p, 4 + i]) - math.sin(a)) < 1e-7


def test_public_names():
    import xdna_engine_b200 as X
    for n in ("PagedCache", "process_logits", "rmsnorm_residual_i8", "rope_table"):
        assert callable(getattr(X, n))
    with pytest.raises(AttributeError):
        X.no_such_name
