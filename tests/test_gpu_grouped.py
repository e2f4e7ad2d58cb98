"""GPU tests of the grouped products (gp_amd/csrc/grouped.hip) against plain 64-bit products.

Every buffer is a view into a larger one filled with NaN (rows before and behind, columns beside): a read outside the
operands reaches a result, a write outside the result is seen."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import grouped_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


def _lib():
    from gp_amd import lib
    return lib


def framed(t, pad, shift):
    """t inside a NaN-filled buffer: `pad` more elements a row, `shift` elements of offset, NaN rows around."""
    *lead, rows, cols = t.shape
    count = int(np.prod(lead)) if lead else 1
    ld = cols + pad
    flat = torch.full((shift + (count * rows + 4) * ld + 8,), float("nan"), dtype=t.dtype, device=t.device)
    view = flat[shift + 2 * ld:shift + 2 * ld + count * rows * ld].view(*lead, rows, ld)[..., :cols]
    view.copy_(t)
    return flat, view


def untouched(flat, view):
    """Everything of the buffer but the view is still NaN."""
    keep = flat.clone()
    inside = keep.as_strided(view.shape, view.stride(), view.storage_offset())
    inside.fill_(float("nan"))
    return bool(torch.isnan(keep).all())


def table(sizes, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(sizes)]), dtype=torch.int64, device="cuda")


def data(seed, dtype, *shape):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float64).to(dtype)


def check(got, want, tol, what=""):
    assert torch.isfinite(got.double()).all(), what
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() - tol).max()))


SHAPES = [
    # sizes of the groups, first row, rows behind the last one, N, K
    ([1], 0, 0, 1, 1),
    ([1], 0, 0, 64, 64),
    ([3, 0, 1], 0, 0, 17, 5),
    ([0, 0, 7, 0], 2, 3, 33, 100),
    ([1, 1, 1, 1, 0, 1, 2], 0, 1, 520, 264),
    ([130, 0, 257, 1], 0, 5, 136, 200),
    ([129, 128, 127], 5, 0, 256, 128),
    ([5, 300], 0, 0, 131, 333),
    ([1] * 70 + [40], 0, 0, 40, 72),
    ([0, 0, 1000], 0, 24, 264, 520),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("w_kc", [True, False], ids=["kc", "nc"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"g{len(s[0])}r{sum(s[0])}n{s[3]}k{s[4]}")
@pytest.mark.parametrize("frame", [(0, 0), (8, 16), (3, 1)], ids=["plain", "aligned", "odd"])
def test_grouped_gemm(dtype, w_kc, shape, frame):
    lib = _lib()
    sizes, first, tail, n, k = shape
    rows = first + sum(sizes) + tail
    x = framed(data(1, dtype, rows, k), *frame)[1]
    x[:first], x[rows - tail:] = float("nan"), float("nan")   # rows of no group are not read
    w = framed(data(2, dtype, len(sizes), *((n, k) if w_kc else (k, n))), *frame)[1]
    old = data(3, dtype, rows, n)
    off = table(sizes, first)
    for alpha, beta in ((1.0, 0.0), (-0.5, 2.0)):
        flat, out = framed(old, *frame)
        if beta == 0.0:
            out[first:rows - tail] = float("nan")   # not read
        assert lib.grouped_gemm(x, w, off, out, w_kc=w_kc, alpha=alpha, beta=beta) is out
        want, tol = oracle.grouped(x.nan_to_num(), w, off.tolist(), old, w_kc, alpha, beta)
        check(out, want, tol, (alpha, beta))
        assert torch.equal(out[:first], old[:first]) and torch.equal(out[rows - tail:], old[rows - tail:])
        assert untouched(flat, out)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("out32", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"g{len(s[0])}r{sum(s[0])}n{s[3]}k{s[4]}")
@pytest.mark.parametrize("frame", [(0, 0), (8, 16), (3, 1)], ids=["plain", "aligned", "odd"])
def test_grouped_gemm_dw(dtype, out32, shape, frame):
    lib = _lib()
    if out32 and dtype == torch.float64:
        return   # refused, see test_refusals
    sizes, first, tail, n, k = shape
    rows = first + sum(sizes) + tail
    x, dy = framed(data(1, dtype, rows, k), *frame)[1], framed(data(2, dtype, rows, n), *frame)[1]
    for t in (x, dy):
        t[:first], t[rows - tail:] = float("nan"), float("nan")
    old = data(3, torch.float32 if out32 else dtype, len(sizes), n, k)
    off = table(sizes, first)
    for alpha, beta in ((1.0, 0.0), (-0.5, 2.0)):
        flat, out = framed(old, *frame)
        if beta == 0.0:
            out.fill_(float("nan"))
        lib.grouped_gemm_dw(x, dy, off, out, alpha=alpha, beta=beta)
        want, tol = oracle.grouped_dw(x.nan_to_num(), dy.nan_to_num(), off.tolist(), old, alpha, beta)
        check(out, want, tol, (alpha, beta))
        assert untouched(flat, out)


RAGGED = [int(v) for v in np.random.RandomState(3).randint(0, 170, 70)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("w_kc", [True, False], ids=["kc", "nc"])
@pytest.mark.parametrize("sizes,n,k", [(RAGGED, 2104, 72), ([9000, 0, 7001, 3999], 1304, 64), ([5000, 300], 264, 520), ([700] * 9, 2056, 136),
                                       ([200] * 40, 520, 264)], ids=["g70", "g4", "g2", "g9", "g40"])
def test_grouped_gemm_on_a_full_chip(dtype, w_kc, sizes, n, k):
    """More tiles than the chip holds at a time, in every tile size and order, more than 64 groups."""
    lib = _lib()
    first, tail = 3, 9
    rows = first + sum(sizes) + tail
    x, w = data(1, dtype, rows, k), data(2, dtype, len(sizes), *((n, k) if w_kc else (k, n)))
    off = table(sizes, first)
    flat, out = framed(torch.full((rows, n), 5.0, dtype=dtype, device="cuda"), 8, 16)
    lib.grouped_gemm(x, w, off, out, w_kc=w_kc)
    want, tol = oracle.grouped(x, w, off.tolist(), torch.full((rows, n), 5.0, dtype=dtype, device="cuda"), w_kc)
    check(out, want, tol)
    assert untouched(flat, out)
    c = lib.grouped_gemm_dw(x, out, off, torch.empty(len(sizes), n, k, dtype=dtype, device="cuda"), alpha=0.25)
    check(c, *oracle.grouped_dw(x, out, off.tolist(), torch.zeros_like(c), alpha=0.25))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("w_kc", [True, False], ids=["kc", "nc"])
@pytest.mark.parametrize("sizes,wide", [([4300], 2000), ([2100, 0, 2290], 2008), ([700, 900, 1300, 1210, 33], 1960)], ids=["g1", "g3", "g5"])
def test_rest_of_a_round(dtype, w_kc, sizes, wide):
    """A few tiles more than whole rounds of the chip, which are done in smaller ones; beta, ragged last tiles."""
    lib = _lib()
    n, k = (2 * wide, 2304) if dtype.itemsize == 2 else (wide, 512)
    rows = 5 + sum(sizes) + 7
    x, w = data(1, dtype, rows, k), data(2, dtype, len(sizes), *((n, k) if w_kc else (k, n)))
    off, old = table(sizes, 5), data(3, dtype, rows, n)
    flat, out = framed(old, 8, 16)
    lib.grouped_gemm(x, w, off, out, w_kc=w_kc, alpha=0.5, beta=-1.0)
    check(out, *oracle.grouped(x, w, off.tolist(), old, w_kc, 0.5, -1.0))
    assert torch.equal(out[:5], old[:5]) and torch.equal(out[rows - 7:], old[rows - 7:]) and untouched(flat, out)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32], ids=str)
@pytest.mark.parametrize("w_kc", [True, False], ids=["kc", "nc"])
@pytest.mark.parametrize("sizes,n,k", [([20000, 0, 31, 15000, 4997], 256, 50), ([33, 40000], 1000, 8), ([30001, 9000], 264, 64), ([40000, 1], 320, 32),
                                       ([513] * 80, 256, 20)], ids=str)
def test_short_k(dtype, w_kc, sizes, n, k):
    """k of at most 512 bytes and many rows: inputs of a few dozen dimensions."""
    lib = _lib()
    k += k if dtype == torch.float32 else 0
    rows = 2 + sum(sizes) + 7
    x, w = framed(data(1, dtype, rows, k), 8, 16)[1], data(2, dtype, len(sizes), *((n, k) if w_kc else (k, n)))
    off, old = table(sizes, 2), data(3, dtype, rows, n)
    for alpha, beta in ((1.0, 0.0), (-0.5, 2.0)):
        flat, out = framed(old, 8, 16)
        lib.grouped_gemm(x, w, off, out, w_kc=w_kc, alpha=alpha, beta=beta)
        check(out, *oracle.grouped(x, w, off.tolist(), old, w_kc, alpha, beta), what=(alpha, beta))
        assert torch.equal(out[:2], old[:2]) and torch.equal(out[rows - 7:], old[rows - 7:]) and untouched(flat, out)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes,n,k", [([9000], 24, 40), ([1, 6000, 0, 2049, 700], 65, 130), ([0, 0, 5000, 0], 130, 17), ([64] * 70 + [8192], 16, 16),
                                       ([20000, 3], 200, 264)], ids=str)
def test_grouped_gemm_dw_over_many_rows(dtype, sizes, n, k):
    """Few results from many rows: the rows are cut into parts whose sums are added afterwards."""
    lib = _lib()
    rows = sum(sizes)
    x, dy = framed(data(1, dtype, rows, k), 3, 1)[1], framed(data(2, dtype, rows, n), 8, 16)[1]
    off = table(sizes)
    for alpha, beta in ((1.0, 0.0), (-0.5, 2.0)):
        old = data(3, dtype, len(sizes), n, k)
        flat, out = framed(old, 3, 1)
        lib.grouped_gemm_dw(x, dy, off, out, alpha=alpha, beta=beta)
        want, tol = oracle.grouped_dw(x, dy, off.tolist(), old, alpha, beta)
        check(out, want, tol, (alpha, beta))
        assert untouched(flat, out)
        again = old.clone()
        lib.grouped_gemm_dw(x, dy, off, again, alpha=alpha, beta=beta)
        assert torch.equal(again, out)
    if dtype in (torch.bfloat16, torch.float16):
        c = lib.grouped_gemm_dw(x, dy, off, torch.empty(len(sizes), n, k, device="cuda"))
        check(c, *oracle.grouped_dw(x, dy, off.tolist(), torch.zeros_like(c)))


def test_wrong_tables_with_many_rows():
    """Tables whose groups overlap name more rows than there are: the result is wrong, nothing outside it is touched."""
    lib = _lib()
    rows, n, k = 9000, 24, 40
    x, dy = data(1, torch.float32, rows, k), data(2, torch.float32, rows, n)
    for offsets in ([0, rows, 0, rows, 0, rows, 0, rows], [rows, -5, 1 << 40, 3, rows, 0, 1, 2]):
        flat, out = framed(torch.zeros(7, n, k, device="cuda"), 8, 16)
        lib.grouped_gemm_dw(x, dy, torch.tensor(offsets, device="cuda"), out)
        assert untouched(flat, out)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_neighbouring_groups_do_not_mix(dtype):
    """NaN in one group's rows stays in that group's results, for row counts on both sides of a tile's edge."""
    lib = _lib()
    for sizes in ([130, 3, 255], [1, 64, 1], [16, 16, 16]):
        rows, n, k = sum(sizes), 72, 40
        x, w, dy = data(1, dtype, rows, k), data(2, dtype, 3, n, k), data(3, dtype, rows, n)
        x[sizes[0]:sizes[0] + sizes[1]] = float("nan")
        off = table(sizes)
        y = lib.grouped_gemm(x, w, off, torch.empty(rows, n, dtype=dtype, device="cuda"))
        c = lib.grouped_gemm_dw(x, dy, off, torch.empty(3, n, k, dtype=dtype, device="cuda"))
        bad = torch.isnan(y).any(1).tolist()
        assert bad == [sizes[0] <= t < sizes[0] + sizes[1] for t in range(rows)]
        assert torch.isnan(c).flatten(1).any(1).tolist() == [False, True, False]


def test_infinite_weights_pass_through():
    """inf * 1 is inf, not NaN, in every type; the padding of k meets no infinity."""
    lib = _lib()
    for dtype in TYPES:
        x = torch.ones(3, 5, dtype=dtype, device="cuda")
        w = torch.ones(1, 4, 5, dtype=dtype, device="cuda")
        w[0, 2, 4] = float("inf")
        y = lib.grouped_gemm(x, w, table([3]), torch.empty(3, 4, dtype=dtype, device="cuda"))
        assert y.tolist() == [[5.0, 5.0, float("inf"), 5.0]] * 3


def test_no_rows_no_columns_no_groups():
    lib = _lib()
    for dtype in TYPES:
        e = lambda *s: torch.full(s, 7.0, dtype=dtype, device="cuda")  # noqa: E731
        assert lib.grouped_gemm(e(0, 8), e(2, 4, 8), table([0, 0]), e(0, 4)).shape == (0, 4)
        assert lib.grouped_gemm(e(3, 8), e(1, 0, 8), table([3]), e(3, 0)).shape == (3, 0)
        assert lib.grouped_gemm(e(3, 8), e(0, 4, 8), table([]), e(3, 4)).tolist() == [[7.0] * 4] * 3
        assert lib.grouped_gemm(e(3, 0), e(1, 4, 0), table([2]), e(3, 4)).tolist() == [[0.0] * 4] * 2 + [[7.0] * 4]
        assert lib.grouped_gemm(e(3, 0), e(1, 4, 0), table([2]), e(3, 4), beta=0.5).tolist() == [[3.5] * 4] * 2 + [[7.0] * 4]
        assert lib.grouped_gemm_dw(e(0, 8), e(0, 4), table([0, 0]), e(2, 4, 8)).tolist() == [[[0.0] * 8] * 4] * 2
        assert lib.grouped_gemm_dw(e(0, 8), e(0, 4), table([0, 0]), e(2, 4, 8), beta=2.0).tolist() == [[[14.0] * 8] * 4] * 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_one_weight_for_all_groups_and_equal_operands(dtype):
    """stride 0 between the groups' weights; X == dY (Gram matrices)."""
    lib = _lib()
    sizes, n, k = [5, 140, 9], 48, 96
    x, w = data(1, dtype, sum(sizes), k), data(2, dtype, 1, n, k).expand(3, n, k)
    out = lib.grouped_gemm(x, w, table(sizes), torch.empty(sum(sizes), n, dtype=dtype, device="cuda"))
    check(out, *oracle.grouped(x, w, table(sizes).tolist(), torch.zeros_like(out)))
    c = lib.grouped_gemm_dw(x, x, table(sizes), torch.empty(3, k, k, dtype=dtype, device="cuda"))
    check(c, *oracle.grouped_dw(x, x, table(sizes).tolist(), torch.zeros_like(c)))
    assert torch.equal(c, c.transpose(1, 2))


@pytest.mark.parametrize("offsets", [[-5, 3, 2, 9, 400], [0, 300, -7, 5, 5], [1 << 40, 4, 2, 1, 0]])
def test_wrong_tables_stay_inside_the_buffers(offsets):
    """Ends outside [0, T] are taken as the nearer end, decreasing pairs as empty groups."""
    lib = _lib()
    rows, n, k = 20, 24, 40
    x, w = framed(data(1, torch.bfloat16, rows, k), 8, 16)[1], data(2, torch.bfloat16, 4, n, k)
    off = torch.tensor(offsets, dtype=torch.int64, device="cuda")
    flat, out = framed(torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda"), 8, 16)
    lib.grouped_gemm(x, w, off, out)
    assert untouched(flat, out)
    reach = oracle.spans(offsets, rows)
    if sum(b - a for a, b in reach) <= rows:   # no row in two groups
        check(out, *oracle.grouped(x, w, offsets, torch.zeros_like(out)))
    c = lib.grouped_gemm_dw(x, x, off, torch.empty(4, k, k, dtype=torch.bfloat16, device="cuda"))
    check(c, *oracle.grouped_dw(x, x, offsets, torch.zeros_like(c)))


def test_offsets_past_32_bits():
    """Rows whose element numbers pass 2^31: the last rows of a 2.3e9-element operand."""
    lib = _lib()
    rows, n, k = 140_000, 24, 16_384
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-300:] = data(1, torch.bfloat16, 300, k)
    w = data(2, torch.bfloat16, 2, n, k)
    off = table([rows - 200, 200])
    out = lib.grouped_gemm(x, w, off, torch.empty(rows, n, dtype=torch.bfloat16, device="cuda"))
    want, tol = oracle.grouped(x[-300:], w, [0, 100, 300], torch.zeros(300, n, dtype=torch.bfloat16, device="cuda"))
    check(out[-300:], want, tol)
    assert not bool(out[:-300].any())
    dy = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    dy[-300:] = data(3, torch.bfloat16, 300, n)
    c = lib.grouped_gemm_dw(x, dy, off, torch.empty(2, n, k, dtype=torch.float32, device="cuda"))
    want, tol = oracle.grouped_dw(x[-300:], dy[-300:], [0, 100, 300], torch.zeros_like(c))
    check(c, want, tol)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_against_differences(dtype):
    """L = sum(R * Y): dx and dw against central differences of L (exact for a bilinear L, up to rounding)."""
    lib = _lib()
    sizes, n, k = [3, 0, 6], 10, 12
    rows = sum(sizes)
    x, w, r = (data(s, dtype, *shape) for s, shape in ((1, (rows, k)), (2, (3, n, k)), (3, (rows, n))))
    off = table(sizes)
    dx = lib.grouped_gemm(r, w, off, torch.empty_like(x), w_kc=False)
    dw = lib.grouped_gemm_dw(x, r, off, torch.empty_like(w))

    def loss(x, w):   # in double through the same entry point
        y = lib.grouped_gemm(x, w, off, torch.empty(rows, n, dtype=torch.float64, device="cuda"))
        return float((y * r.double()).sum())
    h, x, w = 2.0 ** -10, x.double(), w.double()
    half = 2 * oracle.HALF[dtype]
    for at in [(0, 0), (2, 11), (8, 5)]:
        e = torch.zeros_like(x)
        e[at] = h
        d = (loss(x + e, w) - loss(x - e, w)) / (2 * h)
        assert abs(float(dx[at]) - d) <= half * abs(d) + 2e-5 * n
    for at in [(0, 0, 0), (2, 9, 11), (1, 4, 4)]:
        e = torch.zeros_like(w)
        e[at] = h
        d = (loss(x, w + e) - loss(x, w - e)) / (2 * h)
        assert abs(float(dw[at]) - d) <= half * abs(d) + 2e-5 * rows


def test_layouts_agree_with_exchanged_operands():
    """dW of the (G, K, N) layout is the call with x and dy exchanged."""
    lib = _lib()
    sizes, n, k = [30, 7], 24, 56
    x, dy = data(1, torch.float32, 37, k), data(2, torch.float32, 37, n)
    a = lib.grouped_gemm_dw(x, dy, table(sizes), torch.empty(2, n, k, device="cuda"))
    b = lib.grouped_gemm_dw(dy, x, table(sizes), torch.empty(2, k, n, device="cuda"))
    check(a.transpose(1, 2), *oracle.grouped_dw(dy, x, table(sizes).tolist(), torch.zeros_like(b)))
    check(b, *oracle.grouped_dw(dy, x, table(sizes).tolist(), torch.zeros_like(b)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_same_call_same_bits_and_other_streams(dtype):
    lib = _lib()
    sizes, n, k = [200, 0, 700, 1], 200, 136
    x, w, dy = data(1, dtype, 901, k), data(2, dtype, 4, n, k), data(3, dtype, 901, n)
    off = table(sizes)
    run = lambda: (lib.grouped_gemm(x, w, off, torch.empty(901, n, dtype=dtype, device="cuda")),  # noqa: E731
                   lib.grouped_gemm_dw(x, dy, off, torch.empty_like(w)))
    y, c = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:   # two calls at once
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for y2, c2 in got:
        assert torch.equal(y, y2) and torch.equal(c, c2)


def test_captured_and_replayed():
    """A graph of forward, input gradient and weight gradient, replayed on new inputs and offsets beside eager calls."""
    lib = _lib()
    rows, n, k, groups = 600, 136, 200, 3
    x, w, dy = data(1, torch.bfloat16, rows, k), data(2, torch.bfloat16, groups, n, k), data(3, torch.bfloat16, rows, n)
    off = table([100, 200, 250])
    y, dx = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(x)
    c = torch.zeros(groups, n, k, device="cuda")

    def step():
        lib.grouped_gemm(x, w, off, y)
        lib.grouped_gemm(dy, w, off, dx, w_kc=False)
        lib.grouped_gemm_dw(x, dy, off, c)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed, sizes in ((11, [1, 0, 599]), (12, [300, 300, 0]), (13, [0, 0, 0]), (14, [599, 1, 0])):
        x.copy_(data(seed, torch.bfloat16, rows, k))
        off.copy_(table(sizes))
        for t in (y, dx, c):
            t.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, dx, c)]
        for t in (y, dx, c):
            t.fill_(3.0)
        step()
        for a, b in zip(got, (y, dx, c)):
            assert torch.equal(a, b)
        check(y, *oracle.grouped(x, w, off.tolist(), torch.full_like(y, 3.0)))


def test_refusals():
    lib = _lib()
    e = lambda *s, dtype=torch.float32, dev="cuda": torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    x, w, y, off = e(4, 8), e(2, 6, 8), e(4, 6), table([2, 2])
    for bad in (
        lambda: lib.grouped_gemm(x.cpu(), w, off, y),
        lambda: lib.grouped_gemm(x, w.cpu(), off, y),
        lambda: lib.grouped_gemm(x, w, off.cpu(), y),
        lambda: lib.grouped_gemm(x.int(), w.int(), off, y.int()),
        lambda: lib.grouped_gemm(x, w.double(), off, y),
        lambda: lib.grouped_gemm(x, w, off, y.half()),
        lambda: lib.grouped_gemm(x, w, off.int(), y),
        lambda: lib.grouped_gemm(x, w, off[:2], y),
        lambda: lib.grouped_gemm(x, w, e(6, dtype=torch.int64)[::2], y),
        lambda: lib.grouped_gemm(x, w, off, e(4, 7)),
        lambda: lib.grouped_gemm(x, w, off, y, w_kc=False),
        lambda: lib.grouped_gemm(e(8, 4).t(), w, off, y),
        lambda: lib.grouped_gemm(e(1, 8).expand(4, 8), w, off, y),
        lambda: lib.grouped_gemm(x, e(6, 8), off, y),
        lambda: lib.grouped_gemm_dw(x, e(4, 6), off, e(2, 6, 8, dtype=torch.float64)),
        lambda: lib.grouped_gemm_dw(x.double(), e(4, 6).double(), off, e(2, 6, 8)),
        lambda: lib.grouped_gemm_dw(x, e(5, 6), off, e(2, 6, 8)),
        lambda: lib.grouped_gemm_dw(x, e(4, 6), off, e(3, 6, 8)),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(lib.GpxError):   # results of two groups on one another
        lib.grouped_gemm_dw(x, e(4, 6), off, e(1, 6, 8).expand(2, 6, 8))
