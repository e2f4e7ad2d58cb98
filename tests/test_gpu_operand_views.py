"""GPU tests: operands and results that are columns or rows beside one another of one buffer are taken, overlapping ones refused."""
import pytest

torch = pytest.importorskip("torch")
import grouped_oracle as oracle  # noqa: E402
from test_gpu_grouped import check, data, table  # noqa: E402

pytestmark = pytest.mark.gpu


def _lib():
    from gp_amd import lib
    return lib


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_views_of_one_buffer(dtype):
    lib = _lib()
    sizes, n, k = [30, 0, 71], 24, 40
    rows, off = sum(sizes), table([30, 0, 71])
    buf = data(1, dtype, rows, k + n + 8)
    x, y = buf[:, :k], buf[:, k:k + n]
    w = data(2, dtype, 3, n, k)
    want = oracle.grouped(x.clone(), w, off.tolist(), y.clone())
    check(lib.grouped_gemm(x, w, off, y), *want)
    dw = data(3, dtype, 3, 2 * n, k)[:, n:]
    want = oracle.grouped_dw(x, y, off.tolist(), dw.clone())
    check(lib.grouped_gemm_dw(x, y, off, dw), *want)
    stack = data(4, dtype, 3, 2 * n, k)   # the update of the first rows of every matrix into the others
    apart = lib.orthogonalize(stack[:, :n], torch.empty(3, n, k, dtype=dtype, device="cuda"))
    assert torch.equal(lib.orthogonalize(stack[:, :n], stack[:, n:]), apart)


def test_overlaps_are_refused():
    lib = _lib()
    off = table([2, 2])
    buf = torch.zeros(8, 16, device="cuda")
    flat, stack = torch.zeros(1000, device="cuda"), torch.zeros(3, 8, 8, device="cuda")
    w = torch.zeros(2, 8, 8, device="cuda")
    for bad in (lambda: lib.grouped_gemm(buf[:4, :8], w, off, buf[:4, 4:12]),
                lambda: lib.grouped_gemm(buf[:4, :8], w, off, buf[3:7, :8]),
                lambda: lib.grouped_gemm(flat[:32].view(4, 8), w, off, flat[31:63].view(4, 8)),
                lambda: lib.grouped_gemm(buf[:4, :8], w, off, w.view(16, 8)[12:]),
                lambda: lib.grouped_gemm_dw(buf[:4, :8], flat[:32].view(4, 8), off, flat[:128].view(2, 8, 8)),
                lambda: lib.orthogonalize(stack[:2], stack[1:]),
                lambda: lib.orthogonalize(stack[:1].expand(3, 8, 8), stack)):
        with pytest.raises(lib.GpxError):
            bad()


def test_many_groups_of_one_row_and_many_columns():
    """1024 groups of a row and 2^20 columns: in tiles of 32 x 64 these would be more than a launch takes."""
    lib = _lib()
    rows, n, k = 1024, 1 << 20, 16
    x, w = data(1, torch.bfloat16, rows, k), data(2, torch.bfloat16, 1, n, k)
    off = torch.arange(rows + 1, device="cuda")
    y = lib.grouped_gemm(x, w.expand(rows, n, k), off, torch.empty(rows, n, dtype=torch.bfloat16, device="cuda"))
    for at in range(0, n, n // 8):   # sums of 16 products in 32 bits, and the rounding of the result
        cols = slice(at, at + n // 8)
        wt = w[0, cols].double().T.contiguous()
        want, size = x.double() @ wt, x.double().abs() @ wt.abs()
        assert bool(((y[:, cols].double() - want).abs() <= (k + 3) * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all())
