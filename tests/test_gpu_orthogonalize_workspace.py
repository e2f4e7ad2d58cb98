"""GPU test: the workspace that is asked for is what the call uses, on each path of the orthogonalised update."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from test_gpu_grouped import data  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", [(70, 16, 16), (5, 100, 64), (3, 128, 128), (2, 128, 1300), (3, 2100, 40), (24, 50, 8000), (2, 300, 140), (1, 257, 520)], ids=str)
def test_nothing_behind_the_workspace_is_touched(dtype, size):
    from gp_amd import lib
    g = data(1, dtype, *size)
    batch, rows, cols = size
    code = {torch.float64: lib.F64, torch.float32: lib.F32, torch.bfloat16: lib.BF16, torch.float16: lib.F16}[dtype]
    n = C.c_int64(-1)
    assert lib.lib.gpx_orthogonalize_work(code, batch, cols, rows, C.byref(n)) == 0
    guard = 1 << 16
    for steps in (0, 1, 5):
        want = lib.orthogonalize(g, torch.empty_like(g), steps=steps)
        room = torch.full((guard + n.value + guard,), 0xA5, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(g)
        status = lib.lib.gpx_orthogonalize(code, batch, cols, rows, g.data_ptr(), cols, rows * cols, steps, None, 1e-7, out.data_ptr(), cols, rows * cols,
                                           room.data_ptr() + guard, n.value, torch.cuda.current_stream().cuda_stream)
        assert status == 0
        assert bool((room[:guard] == 0xA5).all()) and bool((room[guard + n.value:] == 0xA5).all())
        assert torch.equal(out, want)
