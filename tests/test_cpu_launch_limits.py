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


def test_operands_that_reach_past_the_address_space_are_refused():
    """Row number times leading dimension, or group times stride, past 63 bits."""
    t = (1 << 31) - 2048
    assert gemm(dtype=0, T=t, ldx=1 << 32, X=1 << 30, W=1 << 20, off=1 << 24, Y=1 << 28) == 1
    assert gemm(dtype=0, T=t, ldy=1 << 32, X=1 << 30, W=1 << 20, off=1 << 24, Y=1 << 28) == 1
    assert gemm(dtype=0, groups=65535, sw=1 << 48) == 1
    assert dw(dtype=0, cdtype=0, T=t, ldz=1 << 32, X=1 << 30, Z=1 << 20, off=1 << 24, c=1 << 28) == 1
    assert dw(dtype=0, cdtype=0, N=t, ldz=t, ldc=1 << 32, sc=1 << 48) == 1
    assert ortho(dtype=0, batch=65535, sg=1 << 48) == 1
    assert ortho(dtype=0, batch=65535, so=1 << 48) == 1
