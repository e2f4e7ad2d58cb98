"""CPU tests: what the C entries of the grouped products and of the orthogonalised update refuse, before any GPU call."""
import ctypes as C

import numpy as np
import pytest

from gp_amd import lib

P = 1 << 20   # an aligned address that is never touched: every call here is refused or has nothing to do


def gemm(dtype=2, w_kc=1, groups=2, T=4, N=6, K=8, X=P, ldx=8, W=P, ldw=8, sw=48, off=P, Y=P, ldy=6):
    return lib.lib.gpx_grouped_gemm(dtype, w_kc, groups, T, N, K, 1.0, X, ldx, W, ldw, sw, off, 0.0, Y, ldy, None)


def dw(dtype=2, cdtype=2, groups=2, T=4, M=8, N=6, X=P, ldx=8, Z=P, ldz=6, off=P, c=P, ldc=8, sc=48, work=P, size=1 << 30):
    return lib.lib.gpx_grouped_gemm_dw(dtype, cdtype, groups, T, M, N, 1.0, X, ldx, Z, ldz, off, 0.0, c, ldc, sc, work, size, None)


def ortho(dtype=1, batch=2, M=8, N=6, G=P, ldg=8, sg=48, steps=5, coef=None, eps=1e-7, O=P, ldo=8, so=48, work=P, size=1 << 30):  # noqa: E741
    return lib.lib.gpx_orthogonalize(dtype, batch, M, N, G, ldg, sg, steps, coef, eps, O, ldo, so, work, size, None)


@pytest.mark.parametrize("bad", [dict(dtype=4), dict(dtype=-1), dict(groups=-1), dict(groups=65536), dict(T=-1), dict(N=-1), dict(K=-1),
                                 dict(T=1 << 31), dict(N=1 << 31, ldy=1 << 31), dict(K=1 << 31, ldx=1 << 31, ldw=1 << 31), dict(ldx=7),
                                 dict(ldw=7), dict(w_kc=0, ldw=5), dict(ldy=5), dict(sw=-1), dict(X=None), dict(W=None), dict(Y=None),
                                 dict(off=None), dict(X=P + 1), dict(W=P + 1), dict(Y=P + 1), dict(off=P + 4), dict(dtype=0, X=P + 4)], ids=str)
def test_grouped_gemm_refuses(bad):
    assert gemm(**bad) == 1


@pytest.mark.parametrize("bad", [dict(dtype=4), dict(cdtype=3), dict(cdtype=0), dict(dtype=0, cdtype=1), dict(dtype=1, cdtype=2),
                                 dict(groups=-1), dict(groups=65536), dict(T=-1), dict(M=-1), dict(N=-1), dict(T=1 << 31), dict(ldx=7),
                                 dict(ldz=5), dict(ldc=7), dict(sc=-1), dict(sc=47), dict(X=None), dict(Z=None), dict(c=None), dict(off=None),
                                 dict(X=P + 1), dict(c=P + 1), dict(cdtype=1, c=P + 2), dict(off=P + 2), dict(size=-1)], ids=str)
def test_grouped_gemm_dw_refuses(bad):
    assert dw(**bad) == 1


@pytest.mark.parametrize("bad", [dict(dtype=4), dict(dtype=-1), dict(batch=-1), dict(batch=65536), dict(M=-1), dict(N=-1),
                                 dict(M=(1 << 20) + 1, ldg=1 << 21, ldo=1 << 21), dict(ldg=7), dict(ldo=7), dict(sg=-1), dict(so=47),
                                 dict(steps=-1), dict(steps=65), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                                 dict(G=None), dict(O=None), dict(work=None), dict(G=P + 2), dict(O=P + 2), dict(work=P + 8), dict(size=64)], ids=str)
def test_orthogonalize_refuses(bad):
    assert ortho(**bad) == 1


@pytest.mark.parametrize("call,bad", [(gemm, dict(ldx=(1 << 32) + 1)), (gemm, dict(ldw=1 << 62)), (gemm, dict(ldy=1 << 61)), (gemm, dict(sw=1 << 60)),
                                      (dw, dict(N=5, ldc=1 << 62)), (dw, dict(ldx=1 << 61)), (dw, dict(ldz=1 << 61)), (dw, dict(sc=1 << 60)),
                                      (ortho, dict(N=5, ldo=1 << 62)), (ortho, dict(ldg=1 << 61)), (ortho, dict(sg=1 << 60)),
                                      (ortho, dict(so=1 << 60))], ids=str)
def test_strides_whose_products_would_wrap_are_refused(call, bad):
    assert call(**bad) == 1


def test_an_eps_whose_inverse_overflows_is_refused():
    assert ortho(eps=1e-305) == 1
    assert ortho(eps=5e-324) == 1


def test_orthogonalize_refuses_non_finite_coefficients():
    for v in (np.nan, np.inf):
        c = np.array([1.0, 2.0, 3.0, 1.0, v, 3.0])
        assert ortho(steps=2, coef=c.ctypes.data) == 1


def test_nothing_to_do_needs_no_buffers():
    assert gemm(groups=0, X=None, W=None, Y=None, off=None) == 0
    assert gemm(T=0, X=None, Y=None) == 0
    assert gemm(N=0, ldy=0, W=None, Y=None) == 0
    assert dw(groups=0, c=None, off=None) == 0
    assert dw(M=0, ldx=0, ldc=0, c=None) == 0
    assert ortho(batch=0, G=None, O=None, work=None) == 0
    assert ortho(M=0, ldg=0, ldo=0, G=None, O=None, work=None) == 0


def test_workspace_queries():
    n = C.c_int64(-1)
    assert lib.lib.gpx_orthogonalize_work(1, 2, 100, 300, C.byref(n)) == 0 and n.value > 0
    assert ortho(batch=2, M=100, N=300, ldg=100, ldo=100, sg=30000, so=30000, size=n.value - 1) == 1
    one = n.value
    assert lib.lib.gpx_orthogonalize_work(1, 4, 100, 300, C.byref(n)) == 0 and n.value > one
    assert lib.lib.gpx_orthogonalize_work(1, 0, 100, 300, C.byref(n)) == 0 and n.value == 0
    assert lib.lib.gpx_orthogonalize_work(9, 1, 100, 300, C.byref(n)) == 1
    assert lib.lib.gpx_orthogonalize_work(1, 1, 100, 300, None) == 1
    assert lib.lib.gpx_grouped_gemm_dw_work(2, 4, 1000, 64, 64, C.byref(n)) == 0 and n.value >= 0
    assert lib.lib.gpx_grouped_gemm_dw_work(2, -1, 1000, 64, 64, C.byref(n)) == 1
    assert lib.lib.gpx_grouped_gemm_dw_work(2, 4, 1000, 64, 64, None) == 1
    for dtype in range(4):   # what is asked for is enough, one byte less is refused
        assert lib.lib.gpx_grouped_gemm_dw_work(dtype, 1, 1 << 20, 64, 64, C.byref(n)) == 0
        if n.value:
            assert dw(dtype=dtype, cdtype=dtype, groups=1, T=1 << 20, M=64, N=64, ldx=64, ldz=64, ldc=64, size=n.value - 1) == 1
            assert dw(dtype=dtype, cdtype=dtype, groups=1, T=1 << 20, M=64, N=64, ldx=64, ldz=64, ldc=64, work=None) == 1


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    z = torch.zeros
    with pytest.raises(ValueError):
        lib.grouped_gemm(z(4, 8), z(2, 6, 8), z(3, dtype=torch.int64), z(4, 6))
    with pytest.raises(ValueError):
        lib.grouped_gemm_dw(z(4, 8), z(4, 6), z(3, dtype=torch.int64), z(2, 6, 8))
    with pytest.raises(ValueError):
        lib.orthogonalize(z(4, 8), z(4, 8))
