"""CPU tests of what the orthogonalised update refuses and what workspace it asks for."""
import ctypes as C

import pytest

from gp_amd import lib
from test_cpu_grouped_args import ortho


def work(dtype, batch, M, N):
    n = C.c_int64(-1)
    return lib.lib.gpx_orthogonalize_work(dtype, batch, M, N, C.byref(n)), n.value


@pytest.mark.parametrize("dtype", [lib.BF16, lib.F16])
@pytest.mark.parametrize("size", [(1, 65537), (65537, 1), (300, 70000)], ids=str)
def test_16_bit_sides_above_65536_are_refused_by_both_calls(dtype, size):
    m, n = size
    assert ortho(dtype=dtype, batch=1, M=m, N=n, ldg=m, ldo=m, size=1 << 40) == 1
    assert work(dtype, 1, m, n)[0] == 1
    assert work(dtype, 0, m, n) == (0, 0)   # nothing to do
    assert work(lib.F32, 1, m, n)[0] == 0 and work(lib.F64, 1, m, n)[0] == 0


@pytest.mark.parametrize("dtype", [lib.BF16, lib.F16])
def test_16_bit_sides_up_to_65536_are_taken(dtype):
    assert work(dtype, 1, 65536, 1)[0] == 0 and work(dtype, 2, 100, 65536)[0] == 0


def test_workspace_of_small_matrices_is_small():
    """Matrices that one workgroup holds are worked on there: 4096 of 64 x 64 have 64 MB of floats."""
    for dtype in (lib.F32, lib.BF16, lib.F16):
        assert work(dtype, 4096, 64, 64)[1] <= 1 << 20
        assert work(dtype, 65535, 16, 16)[1] <= 1 << 20
        # short sides over many columns: their columns in 4 bytes a value and the sums, once
        status, n = work(dtype, 4, 4000, 50)
        assert status == 0 and n <= 2 * 4 * 4 * 4000 * 64
