"""CPU tests: sizes whose tiles do not fit one launch are refused as unsupported, before any of their kernels is launched."""
from test_cpu_grouped_args import dw, gemm, ortho

FAR = 1 << 56   # an address behind everything else, never touched


def test_grouped_gemm():
    n = (1 << 31) - 2048
    assert gemm(groups=65535, T=65535, N=n, K=8, sw=0, W=1 << 40, off=1 << 45, Y=FAR, ldy=n) == 4


def test_grouped_gemm_dw():
    for dtype in range(4):
        assert dw(dtype=dtype, cdtype=dtype, groups=1, T=1, M=1 << 20, N=1 << 20, X=1 << 30, ldx=1 << 20, Z=1 << 40, ldz=1 << 20, off=1 << 45,
                  c=FAR, ldc=1 << 20, sc=0) == 4


def test_orthogonalize():
    assert ortho(dtype=0, batch=2000, M=1, N=1 << 20, G=1 << 40, ldg=1, sg=1 << 20, O=1 << 50, ldo=1, so=1 << 20, work=FAR, size=1 << 50) == 4
