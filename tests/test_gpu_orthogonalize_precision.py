"""GPU tests of how exactly the orthogonalised update is computed: 22 bits of every iterate on each of its paths (one workgroup
for all steps, chunks of columns with one launch a step, three tiled products a step), and one rounding of the result."""
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
