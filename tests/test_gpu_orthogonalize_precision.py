"""GPU tests of how exactly the orthogonalised update is computed: 22 bits of every iterate on each of its paths (one workgroup
for all steps, chunks of columns with one launch a step, three tiled products a step), and one rounding of the result."""
import math

import pytest

torch = pytest.importorskip("torch")
import grouped_oracle as oracle  # noqa: E402
from test_gpu_grouped import data  # noqa: E402

pytestmark = pytest.mark.gpu


def _lib():
    from gp_amd import lib
    return lib


def exact(g, steps):
    """The definition in 64 bits, on the short side."""
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = (x.T if tall else x).contiguous()
    x = x / (torch.linalg.norm(x) + 1e-7)
    a, b, c = oracle.COEF
    for _ in range(steps):
        p = x @ x.T.contiguous()
        px = p @ x
        x = a * x + b * px + c * (p @ px)
    return x.T if tall else x


def iterates(steps, side):
    """Relative error of the last iterate: a step takes X (in two products), A and the square factor outside of its diagonal with 22
    bits, and leaves out the product of two second planes, 2^-21 / sqrt(3) a time in the mean square; its sum over the long side is
    taken in 32 bits, 32 terms of three products a time, 3 side / 32 roundings of at most 2^-24 of a sum that only grows; a step
    passes an earlier error on without growth once the singular values have come near one."""
    return (4 * steps * 2.0 ** -42 / 3 + (1 + steps * side / 32) * 2.0 ** -48) ** 0.5


def relative(a, want):
    return float(torch.linalg.norm(a.double() - want) / torch.linalg.norm(want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", [(40, 60), (128, 100), (60, 2900), (128, 1300), (300, 140), (300, 2000), (2000, 300), (1024, 2816)], ids=str)
@pytest.mark.parametrize("steps", [1, 5])
def test_16_bit_results_are_rounded_once(dtype, size, steps):
    """An element whose iterate rounds to another neighbour than its exact value is off by at most the rounding of the exact value and
    twice the iterate's error (both neighbours are half a step from the tie between them): so is the whole matrix, norm-wise."""
    lib = _lib()
    g = data(1, dtype, *size)
    want = exact(g, steps)
    off = relative(lib.orthogonalize(g, torch.empty_like(g), steps=steps), want)
    assert off <= relative(want.to(dtype), want) + 2 * iterates(steps, max(size))


def bound(dtype, want, steps, side):
    """With few singular values, or few sums, the iterates' error is no mean any more: four times as much.  Doubles: three sums of at most
    `side` terms a step, each off by at most side 2^-53."""
    if dtype == torch.float64:
        return 3 * steps * side * 2.0 ** -53
    return relative(want.to(dtype), want) + 8 * iterates(steps, side)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", [(24, 50, 8000), (8, 8192, 128), (9, 16384, 1), (1, 128, 9000), (5, 3, 30000), (24, 8000, 33)], ids=str)
def test_short_sides_of_many_columns(dtype, size):
    """Short sides up to 128 that neither one workgroup nor the chunks of columns take: more chunks than the chip holds at a time, or more
    partial sums than are worth reading again."""
    lib = _lib()
    g = data(1, dtype, *size)
    for steps in (1, 2, 5):
        out = lib.orthogonalize(g, torch.empty_like(g), steps=steps)
        for m in (0, size[0] - 1):
            want = exact(g[m], steps)
            assert relative(out[m], want) <= bound(dtype, want, steps, max(size)), (steps, m)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32], ids=str)
@pytest.mark.parametrize("size", [(1, 3, 66000), (2, 3, 66000), (2, 66000, 3)], ids=str)
def test_sides_above_65536(dtype, size):
    lib = _lib()
    g = data(1, dtype, *size)
    out = lib.orthogonalize(g, torch.empty_like(g), steps=2)
    for got, m in zip(out, g):
        want = exact(m, 2)
        assert relative(got, want) <= bound(dtype, want, 2, max(size))


@pytest.mark.parametrize("size", [(60, 2900), (90, 3000), (96, 2000), (2000, 120), (128, 1300), (64, 20), (128, 128)], ids=str)
@pytest.mark.parametrize("steps", [3, 6])
def test_float32_keeps_22_bits_on_short_sides(size, steps):
    """Every number of 32-row blocks of the short side, in chunks of columns and in one workgroup."""
    lib = _lib()
    g = data(1, torch.float32, *size)
    assert relative(lib.orthogonalize(g, torch.empty_like(g), steps=steps), exact(g, steps)) <= iterates(steps, max(size))


@pytest.mark.parametrize("size", [(30, 44), (300, 140), (3, 20000)], ids=str)
@pytest.mark.parametrize("scale", [-1060, -900, -600, -500, 0, 480, 600, 1000], ids=lambda e: f"2^{e}")
@pytest.mark.parametrize("steps", [0, 2])
def test_doubles_of_any_size(size, scale, steps):
    """Squares of doubles may be out of range where the norm is not: the result is that of the matrix and eps times a power of two."""
    lib = _lib()

    def times(t, e):   # t 2^e, where 2^e may be out of range
        return t * 2.0 ** (e // 2) * 2.0 ** (e - e // 2)
    g = data(1, torch.float64, *size).clamp(-3, 3)
    g[0, 0] = g[-1, -1] = 2.0 ** -300   # far from the rest
    g, eps = times(g, scale), 1e-300
    x = times(g, -scale)   # exact
    x = x / (torch.linalg.norm(x) + math.ldexp(eps, -scale))
    tall = size[0] > size[1]
    x = x.T.contiguous() if tall else x
    a, b, c = oracle.COEF
    for _ in range(steps):
        p = x @ x.T.contiguous()
        x = a * x + b * (p @ x) + c * (p @ (p @ x))
    out = lib.orthogonalize(g, torch.empty_like(g), steps=steps, eps=eps)
    assert relative(out, x.T if tall else x) <= (3 * steps + 1) * max(size) * 2.0 ** -53
